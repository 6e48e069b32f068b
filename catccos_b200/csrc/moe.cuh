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
    uint32_t group_in_lanes;         // 1: a group is the experts of group_lanes whole lanes (a power of two)
    uint32_t group_lanes;            // otherwise: lanes that share the scan of a group (a power of two, groups * group_lanes <= 32)
    uint32_t group_shift;            // log2 of group_lanes
    uint32_t vector, bias_vector;    // 1: a lane's logits (biases) are whole and aligned for vector loads
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

template <uint32_t kBytes>
struct VectorOf {
    using type = uint4;
};
template <>
struct VectorOf<2> {
    using type = uint16_t;
};
template <>
struct VectorOf<4> {
    using type = uint32_t;
};
template <>
struct VectorOf<8> {
    using type = uint2;
};

// kVpl consecutive logits from index `at` of a lane that has all of them (vector loads), in fp32
template <uint32_t kVpl, typename T>
__device__ __forceinline__ void load_logits(const void* p, size_t at, float (&l)[kVpl])
{
    constexpr uint32_t kBytes = kVpl * sizeof(T) < 16 ? kVpl * sizeof(T) : 16;
    constexpr uint32_t kEach = kBytes / sizeof(T);
    using Vector = typename VectorOf<kBytes>::type;
    union {
        Vector v;
        uint16_t h[kBytes / 2];
        uint32_t w[(kBytes + 3) / 4];
    } u;
#pragma unroll
    for (uint32_t i = 0; i < kVpl; i += kEach) {
        u.v = *reinterpret_cast<const Vector*>(static_cast<const T*>(p) + at + i);
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            l[i + j] = __uint_as_float(sizeof(T) == 4 ? u.w[j] : (uint32_t)u.h[j] << 16);
        }
    }
}

__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }

template <typename Real>
__device__ __forceinline__ Real minus_infinity()
{
    return -(Real)INFINITY;
}

// Scores of the fast path, exp and quotient by the fast instructions, in units of 2^-23: exp(x) is off by 2 + 1.5 |x| of
// itself.  A sigmoid s = 1 / (1 + exp(-l)) passes on s (1 - s) of that, at most 0.7 over all l, and adds 2 for the sum and the
// quotient.  A softmax p takes 2 + 2 |l - m| of its own term (p |ln p| < 0.37), their mean over the terms in its sum (the
// entropy of 1024, 6.9), half a unit for each of the sum's 37 additions and 2 for the quotient: under 38 p + 1, and two that
// are compared have p + p' <= 1.  So a difference of two is off by 5.4 or 40 units at most (6.5e-7, 4.8e-6), and the addition
// of a bias adds half a unit of |hi| + |lo|.
constexpr float kSigmoidSlack = 7e-7f, kSoftmaxSlack = 5e-6f;

// Whether hi > lo by more than that.
__device__ __forceinline__ bool apart(float hi, float lo, float slack) { return hi - lo > slack * (1.0f + fabsf(hi) + fabsf(lo)); }

__device__ __forceinline__ float fast_exp(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

__device__ __forceinline__ float fast_inverse(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Keys that order like the floats (minus zero and zero are one value).
__device__ __forceinline__ uint32_t ordered_bits(float v)
{
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return (bits >> 31) != 0u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float from_ordered_bits(uint32_t key) { return __uint_as_float((key >> 31) != 0u ? key & 0x7FFFFFFFu : ~key); }

// Which of this lane's experts are in the top_groups best groups.  c[i] is the choice value of expert lane * kVpl + i, minus
// infinity where it may not be chosen; the others are set to that.  `row`: experts values of this warp's shared memory, used
// where groups are not whole lanes.  Returns false where kSlack and a group that is left out may belong above one that is taken:
// a score is off by the errors of its summands, which go by their own sizes (they may cancel), so every group has its own reach.
template <uint32_t kVpl, typename Real, bool kSlack>
__device__ __forceinline__ bool keep_best_groups(const RouteParams& p, Real (&c)[kVpl], Real* row, uint32_t lane, float slack)
{
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const Real none = minus_infinity<Real>();
    const uint32_t mine = lane >> p.group_shift;
    Real a = none, b = none;  // the two best of this lane's share of its group
    auto take = [&](Real v) {
        b = larger(b, smaller(a, v));
        a = larger(a, v);
    };
    if (p.group_in_lanes != 0u) {
        a = c[0];
#pragma unroll
        for (uint32_t i = 1; i < kVpl; ++i) {
            take(c[i]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            if (lane * kVpl + i < p.experts) {
                row[lane * kVpl + i] = c[i];
            }
        }
        __syncwarp();
        if (mine < p.groups) {
            for (uint32_t j = lane & (p.group_lanes - 1u); j < p.group_size; j += p.group_lanes) {
                take(row[mine * p.group_size + j]);
            }
        }
        __syncwarp();
    }
    for (uint32_t d = p.group_lanes / 2u; d > 0; d >>= 1) {
        const Real oa = __shfl_xor_sync(kAll, a, d), ob = __shfl_xor_sync(kAll, b, d);
        b = larger(larger(b, ob), smaller(a, oa));
        a = larger(a, oa);
    }
    const bool two = p.group_best != 1u && b != none;
    const Real score = two ? a + b : a;
    // the lanes of a group share the comparisons with the others (a group of no expert is below all)
    uint32_t rank = 0;
#pragma unroll 2
    for (uint32_t o0 = 0; o0 < p.groups; o0 += p.group_lanes) {
        const uint32_t o = o0 + (lane & (p.group_lanes - 1u));
        const Real other = __shfl_sync(kAll, score, (o << p.group_shift) & 31u);
        rank += o < p.groups && (other > score || (other == score && o < mine)) ? 1u : 0u;
    }
    for (uint32_t d = p.group_lanes / 2u; d > 0; d >>= 1) {
        rank += __shfl_xor_sync(kAll, rank, d);
    }
    const bool taken = mine < p.groups && rank < p.top_groups && a > none;  // a sum in fp32 may pass its range
    if (p.group_in_lanes != 0u) {
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            c[i] = taken ? c[i] : none;
        }
    } else {
        const uint32_t open = __ballot_sync(kAll, taken);
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            const uint32_t g = (lane * kVpl + i) * p.group_inv >> 22;
            c[i] = g < p.groups && ((open >> (g << p.group_shift)) & 1u) != 0u ? c[i] : none;
        }
    }
    if (!kSlack) {
        return true;
    }
    // Half of apart()'s slack for each of two groups, which covers two values there and four here: 84 or 11.7 units of 2^-23 against
    // 42 or 10.8, and 5.9 units of the values' sizes against one (their additions and the sum).  Infinite sizes tell nothing apart.
    const float reach = slack * (1.0f + (float)(two ? fabs(a) + fabs(b) : fabs(a)));
    const uint32_t least = taken ? ordered_bits(fmaxf((float)score - reach, -3.402823466e38f)) : 0xFFFFFFFFu;
    const uint32_t most = mine < p.groups && !taken && a > none ? ordered_bits(fminf((float)score + reach, 3.402823466e38f)) : 0u;
    return __reduce_min_sync(kAll, least) > __reduce_max_sync(kAll, most);
}

// The top_k experts by value, descending, ties to the lower index: lane r gets the r-th (-1: none left).  One expert a round;
// this is the way of 64-bit values, and of logits of which too many are near the border for gather_candidates().
template <uint32_t kVpl, typename Real>
__device__ __forceinline__ int32_t select_one_by_one(const RouteParams& p, Real (&c)[kVpl], uint32_t lane)
{
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const Real none = minus_infinity<Real>();
    int32_t id = -1;
    for (uint32_t r = 0; r < p.top_k; ++r) {
        Real value = c[0];
        uint32_t e = lane * kVpl;
#pragma unroll
        for (uint32_t i = 1; i < kVpl; ++i) {
            if (c[i] > value) {
                value = c[i];
                e = lane * kVpl + i;
            }
        }
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) {
            const Real ov = __shfl_xor_sync(kAll, value, d);
            const uint32_t oe = __shfl_xor_sync(kAll, e, d);
            if (ov > value || (ov == value && oe < e)) {
                value = ov;
                e = oe;
            }
        }
        if (!(value > none)) {
            break;  // nobody left to choose (the same answer for all lanes)
        }
        if (lane == r) {
            id = (int32_t)e;
        }
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            c[i] = lane * kVpl + i == e ? none : c[i];
        }
    }
    return id;
}

// Shared memory of a warp: the experts that may be among the top_k, by index and by rank.
struct RouteCandidates {
    ulonglong2 found[16];  // the value's ordered bits above, and the complement of the expert below: equal values, lower index first
    float2 sorted[33];     // value, expert's bits
};

// Gathers the experts that may be among the top_k (slack > 0: and the next one, and whatever is within slack of them): the
// (top_k + 1)-th largest of the lanes' best values is a bound that as many values reach, where so many lanes have one; those
// that reach it, a dozen or two, go to s.found in the order of their index.  Returns how many (above 32: only 32 are there).
template <uint32_t kVpl>
__device__ __forceinline__ uint32_t gather_candidates(const RouteParams& p, const float (&c)[kVpl], RouteCandidates& s, uint32_t lane,
                                                      float slack)
{
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const float none = minus_infinity<float>();
    float best = c[0];
#pragma unroll
    for (uint32_t i = 1; i < kVpl; ++i) {
        best = fmaxf(best, c[i]);
    }
    const uint32_t wanted = p.top_k + (slack > 0.0f ? 1u : 0u);
    uint32_t key = ordered_bits(best), bound = 0;
#pragma unroll 4
    for (uint32_t r = 0; r < wanted; ++r) {
        bound = __reduce_max_sync(kAll, key);
        key = key == bound ? 0u : key;
    }
    float least = bound == 0u ? none : from_ordered_bits(bound);
    least = fmaxf(least - 2.0f * slack * (1.0f + fabsf(least)), -3.402823466e38f);  // anything but minus infinity
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kVpl; ++i) {
        mine += c[i] >= least ? 1u : 0u;
    }
    uint32_t end = mine;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(kAll, end, d);
        end += lane >= d ? o : 0u;
    }
    const uint32_t count = __shfl_sync(kAll, end, 31);
    unsigned long long* found = reinterpret_cast<unsigned long long*>(s.found);
    if (lane - count < 4u) {
        found[lane] = 0ull;  // the ranking reads four at a time
    }
    if (mine != 0u && end <= 32u) {
        uint32_t at = smem_u32(s.sorted + (end - mine));
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            // a branch around each store took as long as the rest of this
            asm volatile("{.reg .pred take; setp.ge.f32 take, %1, %2; @take st.shared.v2.b32 [%0], {%1, %3}; @take add.u32 %0, %0, 8;}"
                         : "+r"(at)
                         : "f"(c[i]), "f"(least), "f"(__uint_as_float(lane * kVpl + i))
                         : "memory");
        }
    }
    __syncwarp();
    if (lane < count) {
        const float2 v = s.sorted[lane];
        found[lane] = (unsigned long long)ordered_bits(v.x) << 32 | (0xFFFFFFFFu - __float_as_uint(v.y));
    }
    __syncwarp();
    return count;
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
    return from_ordered_bits(__reduce_max_sync(0xFFFFFFFFu, ordered_bits(v)));
}

// exp(l - m) for l <= m; m may be plus infinity, which then takes all
__device__ __forceinline__ float exp_below(float l, float m) { return l == m ? 1.0f : expf(l - m); }

__device__ __forceinline__ double sigmoid_64(float l) { return 1.0 / (1.0 + exp(-(double)l)); }
__device__ __forceinline__ double exp_below_64(float l, float m) { return l == m ? 1.0 : exp((double)l - (double)m); }

// Sum of exp(l - m) over the token's logits (from index `at`), in 64 bits.  These two read the logits again: given the
// caller's registers, every token would have to put them where an address can point.
template <typename LogitT>
__device__ __noinline__ double softmax_sum_64(const RouteParams& p, size_t at, float m, uint32_t lane)
{
    double sum = 0.0;
    for (uint32_t e = lane; e < p.experts; e += 32u) {
        const float l = load_logit<LogitT>(p.logits, at + e);
        sum += l > minus_infinity<float>() ? exp_below_64(l, m) : 0.0;
    }
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    }
    return sum;
}

// The whole choice in 64 bits: where groups are too close, or too many experts near the border.
template <uint32_t kVpl, typename LogitT>
__device__ __noinline__ int32_t choose_in_64_bits(const RouteParams& p, size_t at, float m, double* row, uint32_t lane)
{
    const double sum = p.sigmoid != 0u ? 1.0 : softmax_sum_64<LogitT>(p, at, m, lane);
    double d[kVpl];
    for (uint32_t i = 0; i < kVpl; ++i) {
        const uint32_t e = lane * kVpl + i;
        d[i] = minus_infinity<double>();
        if (e < p.experts) {
            const float l = load_logit<LogitT>(p.logits, at + e), b = p.bias != nullptr ? p.bias[e] : 0.0f;
            if (l > minus_infinity<float>() && b > minus_infinity<float>()) {
                d[i] = (p.sigmoid != 0u ? sigmoid_64(l) : exp_below_64(l, m) / sum) + (double)b;
            }
        }
    }
    if (p.top_groups < p.groups) {
        keep_best_groups<kVpl, double, false>(p, d, row, lane, 0.0f);
    }
    return select_one_by_one<kVpl, double>(p, d, lane);
}

// One warp a token, kVpl consecutive experts a lane; the logits of a token stay in its registers.  An expert whose logit is
// minus infinity or NaN, or whose bias is, may not be chosen.
//
// The values compared are those of 64 bits, at the price of fast fp32: scores that grow with the logit and have nothing added
// are chosen by the logits themselves; the others are computed with the fast exponential and inverse, and where two neighbours
// of the order are closer than such values can tell apart (one token in some hundred), the dozen candidates are computed and
// ordered in fp64, one a lane; where groups are that close, everything is.
// Bound by instructions at large batches (16384 tokens, 256 experts, top_k 8: 11.5 us by the logits, 15.8 with sigmoid, bias and
// 4 of 8 groups; one expert a round of warp-wide reductions, scores by expf and IEEE divisions and everything again in fp64
// where they were close took 17.7 and 38.7), by the chain of warp-wide steps at small ones (16 tokens: 2.1 and 2.7 us).
template <uint32_t kVpl, typename LogitT>
__global__ void __launch_bounds__(32 * kRouteWarps) moe_route_kernel(const RouteParams p)
{
    extern __shared__ double route_smem[];
    __shared__ RouteCandidates candidates[kRouteWarps];
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t token = blockIdx.x * kRouteWarps + warp;
    grid_dep_wait();
    grid_dep_launch();
    if (token >= p.tokens) {
        return;
    }
    double* row = route_smem + (size_t)warp * p.experts;  // only touched where groups are left out
    RouteCandidates& s = candidates[warp];
    const float none = minus_infinity<float>();
    const uint32_t e0 = lane * kVpl;
    const size_t at = (size_t)token * p.experts;
    const bool by_logit = p.bias == nullptr && (p.top_groups == p.groups || p.group_best == 1u);

    float l[kVpl];
    if (p.vector != 0u && e0 < p.experts) {
        load_logits<kVpl, LogitT>(p.logits, at + e0, l);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            l[i] = e0 + i < p.experts ? load_logit<LogitT>(p.logits, at + e0 + i) : none;
        }
    }
    float m = 0.0f, sum = 1.0f;  // of the softmax; the sum where the weights need it
    if (p.sigmoid == 0u) {
        m = none;
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            m = fmaxf(m, l[i]);
        }
        m = warp_max(m);
        if (p.renormalize == 0u) {
            float part = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                part += l[i] > none ? exp_below(l[i], m) : 0.0f;
            }
            sum = warp_sum(part);
        }
    }

    float c[kVpl];
    float slack = 0.0f;
    bool sure = true;
    if (by_logit) {
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            c[i] = fmaxf(l[i], none);  // NaN becomes minus infinity
        }
        if (p.top_groups < p.groups) {
            keep_best_groups<kVpl, float, false>(p, c, reinterpret_cast<float*>(row), lane, 0.0f);
        }
    } else {
        if (p.sigmoid != 0u) {
            slack = kSigmoidSlack;
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                c[i] = fast_inverse(1.0f + fast_exp(-l[i]));
            }
        } else {
            slack = kSoftmaxSlack;
            float total = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                c[i] = l[i] == m ? 1.0f : fast_exp(l[i] - m);
                total += l[i] > none ? c[i] : 0.0f;
            }
            const float inv = fast_inverse(warp_sum(total));
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                c[i] *= inv;
            }
        }
        float b[kVpl];
        if (p.bias_vector != 0u && e0 < p.experts) {
            load_logits<kVpl, float>(p.bias, e0, b);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kVpl; ++i) {
                b[i] = p.bias != nullptr && e0 + i < p.experts ? p.bias[e0 + i] : 0.0f;
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kVpl; ++i) {
            c[i] = fmaxf(l[i] > none ? c[i] + b[i] : none, none);  // a bias of NaN, too
        }
        if (p.top_groups < p.groups) {
            sure = keep_best_groups<kVpl, float, true>(p, c, reinterpret_cast<float*>(row), lane, slack);
        }
    }
    int32_t id = -1;
    uint32_t count = 33;
    if (sure) {
        count = gather_candidates<kVpl>(p, c, s, lane, slack);
    }
    if (count <= 32u) {
        const unsigned long long mark = reinterpret_cast<const unsigned long long*>(s.found)[lane];
        const float2 own = make_float2(from_ordered_bits((uint32_t)(mark >> 32)), __uint_as_float(0xFFFFFFFFu - (uint32_t)mark));
        uint32_t rank = 0;
        for (uint32_t o = 0; o < count; o += 4u) {
            const ulonglong2 a = s.found[o / 2u], b = s.found[o / 2u + 1u];
            rank += (a.x > mark ? 1u : 0u) + (a.y > mark ? 1u : 0u) + (b.x > mark ? 1u : 0u) + (b.y > mark ? 1u : 0u);
        }
        if (lane < count) {
            s.sorted[rank] = own;
        }
        __syncwarp();
        const float2 placed = lane < count ? s.sorted[lane] : make_float2(none, 0.0f);
        id = lane < min(count, p.top_k) ? (int32_t)__float_as_uint(placed.y) : -1;
        if (slack > 0.0f) {
            const bool clear = !(lane < p.top_k && lane + 1u < count) || apart(placed.x, s.sorted[lane + 1u].x, slack);
            if (!__all_sync(kAll, clear)) {
                const double total = p.sigmoid != 0u ? 1.0 : softmax_sum_64<LogitT>(p, at, m, lane);
                double d = minus_infinity<double>();
                if (lane < count) {
                    const uint32_t e = __float_as_uint(own.y);
                    float le = load_logit<LogitT>(p.logits, at + e);
                    d = (p.sigmoid != 0u ? sigmoid_64(le) : exp_below_64(le, m) / total) + (double)(p.bias != nullptr ? p.bias[e] : 0.0f);
                }
                rank = 0;
                for (uint32_t o = 0; o < count; ++o) {
                    const double v = __shfl_sync(kAll, d, o);
                    rank += v > d || (v == d && o < lane) ? 1u : 0u;
                }
                __syncwarp();
                if (lane < count) {
                    s.sorted[rank] = own;
                }
                __syncwarp();
                id = lane < min(count, p.top_k) ? (int32_t)__float_as_uint(s.sorted[lane].y) : -1;
            }
        }
    } else if (by_logit) {
        id = select_one_by_one<kVpl, float>(p, c, lane);
    } else {
        id = choose_in_64_bits<kVpl, LogitT>(p, at, m, row, lane);
    }

    // lane r: the weight of the r-th expert
    const bool chosen = id >= 0;
    const float lc = chosen ? load_logit<LogitT>(p.logits, at + (uint32_t)id) : none;
    float w;
    if (p.sigmoid != 0u) {
        // sigmoid(l) = 1 / (1 + exp(-|l|)) for l > 0, exp(l) / (1 + exp(-|l|)) otherwise.  Renormalised, a common factor drops
        // out: where all chosen logits are negative, exp of the largest, which keeps the sum away from zero.
        const float q = expf(-fabsf(lc));
        const float top = p.renormalize != 0u ? warp_max(lc) : 0.0f;
        const float below = top < 0.0f ? exp_below(lc, top) : q;
        w = __fdividef(lc > 0.0f ? 1.0f : below, 1.0f + q);  // two units in the last place, for divisors like these
    } else {
        w = p.renormalize != 0u ? exp_below(lc, warp_max(lc)) : __fdividef(exp_below(lc, m), sum);
    }
    if (p.renormalize != 0u) {
        w = chosen ? w : 0.0f;
        w = __fdividef(w, warp_sum(w));
    }
    if (lane < p.top_k) {
        const size_t to = (size_t)token * p.top_k + lane;
        p.ids[to] = id;
        p.weights[to] = chosen ? w * p.scale : 0.0f;
    }
}

// ------------------------------------------------------------------------------------------
// rows of the dispatch
// ------------------------------------------------------------------------------------------
constexpr uint32_t kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanMaxExperts = 1024;  // one thread an expert in the scan
constexpr uint32_t kPlanMaxCluster = 16;
constexpr uint32_t kPlanAhead = 8;

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

// The lanes whose e equals this lane's (e below 2^kBits): one ballot a bit.  match.any does this in one instruction and 60
// cycles of the whole SM; with it the plan of 131072 routes over 256 experts took 41 us.
template <uint32_t kBits>
__device__ __forceinline__ uint32_t same_expert(uint32_t e)
{
    uint32_t same = 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t b = 0; b < kBits; ++b) {
        const uint32_t mine = (uint32_t)((int32_t)(e << (31u - b)) >> 31);  // all ones where the bit is set
        same &= ~(__ballot_sync(0xFFFFFFFFu, mine != 0u) ^ mine);
    }
    return same;
}

// A stable counting sort of the routes by expert, in one launch of one CTA or one cluster (the CTAs exchange their counts
// through distributed shared memory; nothing is kept between launches).  Every warp owns a contiguous run of routes and counts
// it in its own row of shared memory; then each route's place is its expert's first row, what the CTAs and warps before hold
// of that expert, and the routes of its own warp in front of it, 32 at a time: the order of the routes, whatever the timing.
template <uint32_t kBits>
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
    const uint32_t busy = min(kPlanWarps, (uint32_t)(((uint64_t)p.routes + p.per_warp - 1u) / p.per_warp));  // warps of a CTA, at most

    for (uint32_t i = threadIdx.x; i < busy * p.experts; i += kPlanThreads) {
        counts[i] = 0u;
    }
    grid_dep_wait();
    grid_dep_launch();
    __syncthreads();

    // kPlanAhead runs of 32 routes at a time, all loads on their way together; a warp that has no more than that keeps them
    uint32_t x[kPlanAhead];
    auto load = [&](uint32_t r) {
        int32_t id[kPlanAhead];
#pragma unroll
        for (uint32_t j = 0; j < kPlanAhead; ++j) {
            id[j] = r + j * 32u + lane < r1 ? p.ids[r + j * 32u + lane] : -1;
        }
#pragma unroll
        for (uint32_t j = 0; j < kPlanAhead; ++j) {
            const uint32_t e = (uint32_t)id[j] - (uint32_t)p.first;
            x[j] = id[j] >= p.first && e < p.experts ? e : p.experts;  // experts: none of this rank's
        }
    };
    for (uint32_t r = r0; r < r1; r += kPlanAhead * 32u) {
        load(r);
#pragma unroll
        for (uint32_t j = 0; j < kPlanAhead; ++j) {
            if (x[j] < p.experts) {
                atomicAdd(mine + x[j], 1u);  // counts do not depend on the order
            }
        }
    }
    __syncthreads();
    // per expert: what the warps before counted, and the CTA's total
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
            uint32_t v[kPlanMaxCluster];
#pragma unroll
            for (uint32_t c = 0; c < kPlanMaxCluster; ++c) {
                v[c] = 0u;
                if (c < ctas) {
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[c]) : "r"(map_to_cta(smem_u32(totals + e), c)) : "memory");
                }
            }
#pragma unroll
            for (uint32_t c = 0; c < kPlanMaxCluster; ++c) {
                before += c < cta ? v[c] : 0u;
                all += v[c];
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

    for (uint32_t r = r0; r < r1; r += kPlanAhead * 32u) {
        if (r1 - r0 > kPlanAhead * 32u) {
            load(r);
        }
#pragma unroll
        for (uint32_t j = 0; j < kPlanAhead; ++j) {
            if (r + j * 32u >= r1) {
                break;
            }
            const bool has = x[j] < p.experts;
            const uint32_t same = same_expert<kBits>(x[j]) & __ballot_sync(kAll, has);
            const uint32_t ahead = (uint32_t)__popc(same & ((1u << lane) - 1u));
            const uint32_t at = has ? mine[x[j]] : 0u;
            __syncwarp();
            if (has && ahead == 0u) {
                mine[x[j]] = at + (uint32_t)__popc(same);
            }
            __syncwarp();
            if (r + j * 32u + lane < r1) {
                p.row_index[r + j * 32u + lane] = has ? (int32_t)(begin[x[j]] + at + ahead) : -1;
            }
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
    uint32_t vectors;          // lanes of a token: n / 8, or n / 16 in the wide form
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
// Bound by memory: every live row once, 2 n bytes, and the result.  A lane owns eight columns of a token and has up to eight
// rows on their way before it adds the first, or (wide) sixteen columns, a whole sector a load, and four rows.  4095 tokens x 8
// rows of 7168 columns: 79 us wide (6.5 TB/s), 97 to 106 narrow; 16 tokens, where one round trip counts: see combine_wide().
template <typename T, bool kWide>
__global__ void __launch_bounds__(kCombineThreads, kWide ? 7 : 1) moe_combine_kernel(const CombineParams p)
{
    constexpr uint32_t kWords = kWide ? 8 : 4, kInFlight = kWide ? 4 : 8;
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
    auto load = [&](const uint8_t* base, size_t row, uint32_t (&x)[kWords]) {
        const uint8_t* src = base + (row * p.vectors + v) * (kWords * 4u);
        uint4 a, b;
        if constexpr (kWide) {
            ld_global_stream_v8(src, a, b);
            x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            a = __ldcs(reinterpret_cast<const uint4*>(src));
        }
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    };
    float acc[2 * kWords] = {};
    for (uint32_t r0 = 0; r0 < p.top_k; r0 += kInFlight) {
        uint32_t index[kInFlight];
        float w[kInFlight];
        uint32_t row[kInFlight][kWords];
        bool live[kInFlight];
        // all indices before the first row: one round trip for them, one for the rows
#pragma unroll
        for (uint32_t j = 0; j < kInFlight; ++j) {
            const size_t at = (size_t)token * p.top_k + min(r0 + j, p.top_k - 1u);
            index[j] = (uint32_t)__ldcg(p.row_index + at);
            w[j] = __ldcg(p.weights + at);
        }
#pragma unroll
        for (uint32_t j = 0; j < kInFlight; ++j) {
            live[j] = r0 + j < p.top_k && index[j] < p.rows;  // a dropped route is negative: above any row
#pragma unroll
            for (uint32_t i = 0; i < kWords; ++i) {
                row[j][i] = 0u;
            }
            if (live[j]) {
                load(p.y, index[j], row[j]);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kInFlight; ++j) {
            if (live[j]) {
#pragma unroll
                for (uint32_t i = 0; i < kWords; ++i) {
                    const float2 f = unpack2<T>(row[j][i]);
                    acc[2 * i] = fmaf(w[j], f.x, acc[2 * i]);
                    acc[2 * i + 1] = fmaf(w[j], f.y, acc[2 * i + 1]);
                }
            }
        }
    }
    if (p.shared_out != nullptr) {
        uint32_t x[kWords];
        load(p.shared_out, token, x);
#pragma unroll
        for (uint32_t i = 0; i < kWords; ++i) {
            const float2 f = unpack2<T>(x[i]);
            acc[2 * i] += f.x;
            acc[2 * i + 1] += f.y;
        }
    }
    uint32_t o[kWords];
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
        o[i] = pack2<T>(acc[2 * i], acc[2 * i + 1]);
    }
    uint8_t* dst = p.out + ((size_t)token * p.vectors + v) * (kWords * 4u);
    if constexpr (kWide) {
        st_global_v8(dst, o);
    } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace catccos
