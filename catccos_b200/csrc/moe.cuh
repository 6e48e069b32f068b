// The mixture-of-experts steps around the experts' products: scores to experts and weights (moe_route_kernel), the rows of the
// dispatch (moe_row_plan_kernel: the expanded_row_idx that mx_quant_scatter_packed_kernel takes, and where each expert's rows
// begin), and the weighted sum of a token's expert rows (moe_combine_kernel).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "mx_gemm.cuh"

namespace catccos {

// ------------------------------------------------------------------------------------------
// routing
// ------------------------------------------------------------------------------------------
constexpr uint32_t kRouteWarps = 4;  // tokens of a CTA
constexpr uint32_t kRouteMaxExperts = 1024, kRouteMaxTopK = 32, kRouteMaxGroups = 32;

struct RouteParams {
    const void* logits;  // fp32 or bf16 [tokens, experts]
    const float* bias;   // [experts] or nullptr
    int32_t* ids;        // [tokens, top_k]
    float* weights;      // [tokens, top_k]
    uint32_t tokens, experts, top_k, groups, top_groups, group_best;
    uint32_t sigmoid, renormalize;
    float scale;
    uint32_t group_size, group_inv;  // experts / groups, and 2^22 / group_size + 1: e / group_size == e * group_inv >> 22 (e < 1024)
    uint32_t group_lanes;            // lanes that share a group's scan (a power of two, groups * group_lanes <= 32)
};

template <typename T>
__device__ __forceinline__ float load_logit(const void* p, size_t i);
template <>
__device__ __forceinline__ float load_logit<float>(const void* p, size_t i)
{
    return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float load_logit<__nv_bfloat16>(const void* p, size_t i)
{
    return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}

template <typename Real>
__device__ __forceinline__ Real minus_infinity()
{
    return -(Real)INFINITY;
}

// What a warp knows about its token's choice after select_experts(): lane r holds the r-th expert (-1: none left), and
// whether every comparison that the choice rests on was wider than `slack`, the error of the values compared.
struct Choice {
    int32_t id;
    bool sure;
};

// The top_k experts of a token by value (descending, ties to the lower index), in its top_groups best groups.  c[i] is the
// value of expert i * 32 + lane, minus infinity where it may not be chosen; c is used up.  `row` is this warp's shared memory
// (experts values).  kSlack false: the values are exact.
template <uint32_t kVpl, typename Real, bool kSlack>
__device__ __forceinline__ Choice select_experts(const RouteParams& p, Real (&c)[kVpl], Real* row, uint32_t lane)
{
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const Real none = minus_infinity<Real>();
    // fp32 scores are off by less than 2^-19 (softmax over 1024 experts: 40 roundings of 2^-24 in the sum, four units in the
    // last place of expf and the division; sigmoid less), sums with a bias by half a unit in their last place more
    auto apart = [](Real hi, Real lo) { return hi - lo > (Real)3.9e-6 * ((Real)1 + (hi < 0 ? -hi : hi) + (lo < 0 ? -lo : lo)); };
    Choice choice = {-1, true};
    if (p.top_groups < p.groups) {
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            if (i * 32u + lane < p.experts) {
                row[i * 32u + lane] = c[i];
            }
        }
        __syncwarp();
        const uint32_t mine = lane / p.group_lanes;
        Real a = none, b = none;  // the two best of this lane's share of its group
        if (mine < p.groups) {
            for (uint32_t j = lane % p.group_lanes; j < p.group_size; j += p.group_lanes) {
                const Real v = row[mine * p.group_size + j];
                b = v > a ? a : (v > b ? v : b);
                a = v > a ? v : a;
            }
        }
        __syncwarp();
        for (uint32_t d = p.group_lanes / 2u; d > 0; d >>= 1) {
            const Real oa = __shfl_xor_sync(kAll, a, d), ob = __shfl_xor_sync(kAll, b, d);
            const Real low = a < oa ? a : oa, second = b > ob ? b : ob;
            a = a > oa ? a : oa;
            b = low > second ? low : second;
        }
        const Real score = p.group_best == 1u || b == none ? a : a + b;
        uint32_t rank = 0;
        for (uint32_t o = 0; o < p.groups; ++o) {
            const Real other = __shfl_sync(kAll, score, o * p.group_lanes);
            rank += other > score || (other == score && o < mine) ? 1u : 0u;
        }
        const bool taken = mine < p.groups && rank < p.top_groups && score > none;
        if (kSlack) {
            // the border: the last group taken against the first one left out
            Real last = taken ? score : -none, first = mine < p.groups && !taken ? score : none;
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) {
                const Real ol = __shfl_xor_sync(kAll, last, d), of = __shfl_xor_sync(kAll, first, d);
                last = ol < last ? ol : last;
                first = of > first ? of : first;
            }
            choice.sure = first == none || last == -none || apart(last * (Real)0.5, first * (Real)0.5);  // sums of two
        }
        const uint32_t open = __ballot_sync(kAll, taken);
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            const uint32_t g = (i * 32u + lane) * p.group_inv >> 22;
            if (g >= p.groups || ((open >> (g * p.group_lanes)) & 1u) == 0u) {
                c[i] = none;
            }
        }
    }
    // one expert a round: every lane keeps the best of its own
    Real best, previous = none;
    uint32_t at;
    auto rescan = [&]() {
        best = c[0];
        at = 0;
#pragma unroll
        for (uint32_t i = 1; i < kVpl; ++i) {
            if (c[i] > best) {
                best = c[i];
                at = i;
            }
        }
    };
    rescan();
    for (uint32_t r = 0; r < p.top_k + (kSlack ? 1u : 0u); ++r) {
        Real value;
        uint32_t e;
        if constexpr (std::is_same<Real, float>::value) {
            const uint32_t bits = __float_as_uint(best + 0.0f);  // minus zero and zero are one value
            const uint32_t key = (bits >> 31) != 0u ? ~bits : bits | 0x80000000u;
            const uint32_t top = __reduce_max_sync(kAll, key);
            e = __reduce_min_sync(kAll, key == top ? at * 32u + lane : 0xFFFFFFFFu);
            value = __uint_as_float((top >> 31) != 0u ? top & 0x7FFFFFFFu : ~top);
        } else {
            value = best;
            e = at * 32u + lane;
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) {
                const Real ov = __shfl_xor_sync(kAll, value, d);
                const uint32_t oe = __shfl_xor_sync(kAll, e, d);
                if (ov > value || (ov == value && oe < e)) {
                    value = ov;
                    e = oe;
                }
            }
        }
        if (!(value > none)) {
            break;  // nobody left to choose (the same answer for all lanes)
        }
        if (kSlack && r > 0u && !apart(previous, value)) {
            choice.sure = false;
            break;
        }
        previous = value;
        if (lane == r) {
            choice.id = (int32_t)e;
        }
        if ((e & 31u) == lane) {
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                if (i == e >> 5) {
                    c[i] = none;
                }
            }
            rescan();
        }
    }
    if (lane >= p.top_k) {
        choice.id = -1;  // the round behind the last one only looks at the distance
    }
    return choice;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
        v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    }
    return v;
}

__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    }
    return v;
}

// exp(l - m) for l <= m; m may be plus infinity, which then takes all
__device__ __forceinline__ float exp_below(float l, float m) { return l == m ? 1.0f : expf(l - m); }

// One warp a token; the logits of a token stay in its registers.  An expert whose logit is minus infinity or NaN, or whose
// bias is, may not be chosen.
//
// The values compared are those of 64 bits, at the price of 32: scores that grow with the logit and have nothing added are
// chosen by the logits themselves; the others are computed in fp32, and where two values that decide the choice are closer
// than fp32 can tell apart (one token in several hundred), the warp does it again in fp64.
// Latency bound up to some thousand tokens: top_k rounds of two warp reductions (redux.sync) each.
template <uint32_t kVpl, typename LogitT>
__global__ void __launch_bounds__(32 * kRouteWarps) moe_route_kernel(const RouteParams p)
{
    extern __shared__ double route_smem[];
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t token = blockIdx.x * kRouteWarps + warp;
    grid_dep_wait();
    grid_dep_launch();
    if (token >= p.tokens) {
        return;
    }
    double* row = route_smem + (size_t)warp * p.experts;  // only touched where groups are left out
    const float none = minus_infinity<float>();

    float l[kVpl];
    float m = none;
#pragma unroll
    for (uint32_t i = 0; i < kVpl; ++i) {
        const uint32_t e = i * 32u + lane;
        l[i] = none;
        if (e < p.experts) {
            l[i] = load_logit<LogitT>(p.logits, (size_t)token * p.experts + e);
            l[i] = l[i] > none ? l[i] : none;  // NaN
        }
        m = fmaxf(m, l[i]);
    }
    float sum = 1.0f;
    if (p.sigmoid == 0u) {
        m = warp_max(m);
        float part = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            part += l[i] > none ? exp_below(l[i], m) : 0.0f;
        }
        sum = warp_sum(part);
    }

    Choice choice;
    if (p.bias == nullptr && (p.top_groups == p.groups || p.group_best == 1u)) {
        float c[kVpl];
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            c[i] = l[i];
        }
        choice = select_experts<kVpl, float, false>(p, c, reinterpret_cast<float*>(row), lane);
    } else {
        float c[kVpl];
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            const uint32_t e = i * 32u + lane;
            const float b = p.bias != nullptr && e < p.experts ? p.bias[e] : 0.0f;
            const float s = p.sigmoid != 0u ? 1.0f / (1.0f + expf(-l[i])) : exp_below(l[i], m) / sum;
            c[i] = l[i] > none && b > none ? s + b : none;
        }
        choice = select_experts<kVpl, float, true>(p, c, reinterpret_cast<float*>(row), lane);
        if (!__all_sync(kAll, choice.sure)) {
            double d[kVpl];
            double part = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                d[i] = 0.0;
                if (l[i] > none) {
                    d[i] = p.sigmoid != 0u ? 1.0 / (1.0 + exp(-(double)l[i])) : (l[i] == m ? 1.0 : exp((double)l[i] - (double)m));
                }
                part += d[i];
            }
#pragma unroll
            for (uint32_t s = 16; s > 0; s >>= 1) {
                part += __shfl_xor_sync(kAll, part, s);
            }
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                const uint32_t e = i * 32u + lane;
                const float b = p.bias != nullptr && e < p.experts ? p.bias[e] : 0.0f;
                const double s = p.sigmoid != 0u ? d[i] : d[i] / part;
                d[i] = l[i] > none && b > none ? s + (double)b : minus_infinity<double>();
            }
            __syncwarp();
            choice = select_experts<kVpl, double, false>(p, d, row, lane);
        }
    }

    // lane r: the weight of the r-th expert
    const bool chosen = choice.id >= 0;
    const float lc = chosen ? load_logit<LogitT>(p.logits, (size_t)token * p.experts + (uint32_t)choice.id) : none;
    float w;
    if (p.renormalize != 0u) {
        // a common factor of the chosen scores drops out: taking the largest logit for it keeps the sum away from zero
        const float top = warp_max(lc);
        if (p.sigmoid != 0u) {
            const float f = fminf(top, 0.0f);
            w = lc > 0.0f ? 1.0f / (1.0f + expf(-lc)) : exp_below(lc, f) / (1.0f + expf(lc));
        } else {
            w = exp_below(lc, top);
        }
        w = chosen ? w : 0.0f;
        w /= warp_sum(w);
    } else {
        w = p.sigmoid != 0u ? 1.0f / (1.0f + expf(-lc)) : exp_below(lc, m) / sum;
    }
    if (lane < p.top_k) {
        const size_t at = (size_t)token * p.top_k + lane;
        p.ids[at] = choice.id;
        p.weights[at] = chosen ? w * p.scale : 0.0f;
    }
}

// ------------------------------------------------------------------------------------------
// rows of the dispatch
// ------------------------------------------------------------------------------------------
constexpr uint32_t kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanMaxExperts = 1024;  // one thread an expert in the scan
constexpr uint32_t kPlanCluster = 8;

struct RowPlanParams {
    const int32_t* ids;   // [routes]
    int32_t* row_index;   // [routes]
    int32_t* offsets;     // [experts + 1]
    uint32_t routes, experts;
    int32_t first;
    uint32_t per_warp;    // routes of a warp, a multiple of 32
};

// [kPlanWarps][experts] counts, [experts] totals of this CTA, [experts] first rows, [32] of the scan
__host__ __device__ constexpr size_t row_plan_smem(uint32_t experts) { return ((size_t)(kPlanWarps + 2) * experts + 32) * 4; }

// A stable counting sort of the routes by expert, in one launch of one CTA or one cluster (the CTAs exchange their counts
// through distributed shared memory; nothing is kept between launches).  Every warp owns a contiguous run of routes and counts
// it in its own row of shared memory, 32 routes at a time: lanes with the same expert find one another (match.any) and the
// lowest adds for all of them, so there is no atomic and the order is that of the routes.
__global__ void __launch_bounds__(kPlanThreads, 1) moe_row_plan_kernel(const RowPlanParams p, uint32_t ctas)
{
    extern __shared__ uint32_t plan_smem[];
    uint32_t* counts = plan_smem;
    uint32_t* totals = counts + kPlanWarps * p.experts;
    uint32_t* begin = totals + p.experts;
    uint32_t* scan = begin + p.experts;
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t cta = blockIdx.x;  // the grid is one cluster
    const uint64_t from = (uint64_t)(cta * kPlanWarps + warp) * p.per_warp;
    const uint32_t r0 = (uint32_t)min(from, (uint64_t)p.routes), r1 = (uint32_t)min(from + p.per_warp, (uint64_t)p.routes);
    uint32_t* mine = counts + warp * p.experts;

    for (uint32_t i = threadIdx.x; i < kPlanWarps * p.experts; i += kPlanThreads) {
        counts[i] = 0u;
    }
    grid_dep_wait();
    grid_dep_launch();
    __syncthreads();

    auto expert_of = [&](uint32_t r) {
        const uint32_t e = r < r1 ? (uint32_t)p.ids[r] - (uint32_t)p.first : 0xFFFFFFFFu;
        return r < r1 && p.ids[r] >= p.first && e < p.experts ? e : 0xFFFFFFFFu;
    };
    for (uint32_t r = r0; r < r1; r += 32u) {
        const uint32_t e = expert_of(r + lane);
        const uint32_t same = __match_any_sync(kAll, e);
        if (e != 0xFFFFFFFFu && lane == (uint32_t)__ffs((int)same) - 1u) {
            mine[e] += (uint32_t)__popc(same);
        }
        __syncwarp();
    }
    __syncthreads();
    // per expert: what the warps before counted, and the CTA's total
    const uint32_t busy = min(kPlanWarps, (uint32_t)(((uint64_t)p.routes + p.per_warp - 1u) / p.per_warp));
    const uint32_t e = threadIdx.x;
    if (e < p.experts) {
        uint32_t run = 0;
        for (uint32_t w = 0; w < busy; ++w) {
            const uint32_t v = counts[w * p.experts + e];
            counts[w * p.experts + e] = run;
            run += v;
        }
        totals[e] = run;
    }
    uint32_t before = 0, all = 0;
    if (ctas > 1u) {
        __syncwarp();
        cluster_sync_all();
        if (e < p.experts) {
            for (uint32_t c = 0; c < ctas; ++c) {
                uint32_t v;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(totals + e), c)) : "memory");
                before += c < cta ? v : 0u;
                all += v;
            }
        }
    } else if (e < p.experts) {
        all = totals[e];
    }
    // exclusive scan over the experts
    uint32_t incl = all;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(kAll, incl, d);
        incl += lane >= d ? o : 0u;
    }
    if (lane == 31u) {
        scan[warp] = incl;
    }
    __syncthreads();
    if (warp == 0) {
        const uint32_t v = scan[lane];
        uint32_t s = v;
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) {
            const uint32_t o = __shfl_up_sync(kAll, s, d);
            s += lane >= d ? o : 0u;
        }
        scan[lane] = s - v;
    }
    __syncthreads();
    if (e < p.experts) {
        const uint32_t first_row = scan[warp] + incl - all;
        begin[e] = first_row + before;
        if (cta == 0) {
            p.offsets[e] = (int32_t)first_row;
            if (e + 1u == p.experts) {
                p.offsets[p.experts] = (int32_t)(first_row + all);
            }
        }
    }
    __syncthreads();

    for (uint32_t r = r0; r < r1; r += 32u) {
        const uint32_t x = expert_of(r + lane);
        const uint32_t same = __match_any_sync(kAll, x);
        const uint32_t ahead = (uint32_t)__popc(same & ((1u << lane) - 1u));
        const uint32_t at = x != 0xFFFFFFFFu ? mine[x] : 0u;
        __syncwarp();
        if (x != 0xFFFFFFFFu && ahead == 0u) {
            mine[x] = at + (uint32_t)__popc(same);
        }
        __syncwarp();
        if (r + lane < r1) {
            p.row_index[r + lane] = x != 0xFFFFFFFFu ? (int32_t)(begin[x] + at + ahead) : -1;
        }
    }
    if (ctas > 1u) {
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another may still read its totals
    }
}

// ------------------------------------------------------------------------------------------
// combine
// ------------------------------------------------------------------------------------------
constexpr uint32_t kCombineThreads = 128;

struct CombineParams {
    const uint8_t* y;          // [rows, n], 16-bit floats
    const int32_t* row_index;  // [tokens, top_k]
    const float* weights;      // [tokens, top_k]
    const uint8_t* shared_out; // [tokens, n] or nullptr
    uint8_t* out;              // [tokens, n]
    uint32_t tokens, rows, n, top_k;
    uint32_t vectors;          // n / 8
    uint32_t slabs;            // CTAs of a token, or 0: a CTA has several tokens
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v)
{
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// out[t] = sum over r of weights[t, r] * y[row_index[t, r]], r ascending, in fp32 (+ shared_out[t]), rounded once.
// Bound by memory: every live row once, 2 n bytes, and the result.  A lane owns eight columns of a token (16-byte loads, whole
// lines a warp) and has up to eight rows on their way before it adds the first.
template <typename T>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const CombineParams p)
{
    constexpr uint32_t kInFlight = 8;
    grid_dep_wait();
    grid_dep_launch();
    uint32_t token, v;
    if (p.slabs != 0u) {
        token = blockIdx.x / p.slabs;
        v = (blockIdx.x - token * p.slabs) * kCombineThreads + threadIdx.x;
    } else {
        const uint32_t in_cta = threadIdx.x / p.vectors;
        token = blockIdx.x * (kCombineThreads / p.vectors) + in_cta;
        v = threadIdx.x - in_cta * p.vectors;
        if (in_cta >= kCombineThreads / p.vectors) {
            return;
        }
    }
    if (token >= p.tokens || v >= p.vectors) {
        return;
    }
    float acc[8] = {};
    for (uint32_t r0 = 0; r0 < p.top_k; r0 += kInFlight) {
        uint4 row[kInFlight];
        float w[kInFlight];
        bool live[kInFlight];
#pragma unroll
        for (uint32_t j = 0; j < kInFlight; ++j) {
            live[j] = false;
            if (r0 + j < p.top_k) {
                const size_t at = (size_t)token * p.top_k + r0 + j;
                const uint32_t index = (uint32_t)__ldcg(p.row_index + at);  // a dropped route is negative: above any row
                live[j] = index < p.rows;
                w[j] = __ldcg(p.weights + at);
                if (live[j]) {
                    row[j] = __ldcs(reinterpret_cast<const uint4*>(p.y) + (size_t)index * p.vectors + v);
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kInFlight; ++j) {
            if (live[j]) {
                const uint32_t x[4] = {row[j].x, row[j].y, row[j].z, row[j].w};
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float2 f = unpack2<T>(x[i]);
                    acc[2 * i] = fmaf(w[j], f.x, acc[2 * i]);
                    acc[2 * i + 1] = fmaf(w[j], f.y, acc[2 * i + 1]);
                }
            }
        }
    }
    const size_t at = (size_t)token * p.vectors + v;
    if (p.shared_out != nullptr) {
        const uint4 s = __ldcs(reinterpret_cast<const uint4*>(p.shared_out) + at);
        const uint32_t x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(x[i]);
            acc[2 * i] += f.x;
            acc[2 * i + 1] += f.y;
        }
    }
    reinterpret_cast<uint4*>(p.out)[at] =
        make_uint4(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]), pack2<T>(acc[4], acc[5]), pack2<T>(acc[6], acc[7]));
}

}  // namespace catccos
