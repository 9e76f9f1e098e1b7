// Routing to experts for models whose routing is neither of clb_route_device's modes: scores
// of three kinds, a bias for balance, groups of experts, top-k, renormalised weights.
//
// Ranks are compared as fp32 values that are the same on every machine: a score is the
// correctly rounded float, the bias is added in fp32, and ties go to the lower id. Without a
// bias the rank is the logit, since every score rises with it. Evaluating every score in
// double costs more than all the rest, so scores are first evaluated in fp32 with a known
// error; if the picks (and the groups) are further apart than that error they are the same
// as with exact scores, else (about one row in a thousand with continuous logits) the experts
// in question are ranked in double.
#include <cfloat>
#include <cmath>

#include "clb_ops.cuh"

namespace clb {
namespace {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxPicks = 16;
constexpr int kRouteMaxGroups = 32;
constexpr int kRouteWarps = 4;
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // rank_key(-inf): an expert that is not available
constexpr float kHalfUlp = 0x1p-24f;

struct RouteArgs {
    const void* logits;
    const float* bias;
    int* ids;
    float* w;
    int* status;
    int64_t ld;
    int tokens, type, E, k, groups, top_groups, pair, renorm;
    int per, log_lanes;  // experts of a group; 2^log_lanes lanes work on one, groups << log_lanes <= 32
    float scale, per_inv;  // per_inv: groups / E
};

// Order-preserving map of a float to unsigned (-0 as +0).
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

// exp(l - top): the rounding of the difference, which the exponential would carry as a relative
// error of |l - top| half ulps, is found exactly (the two-sum of l and -top) and put back.
__device__ __forceinline__ float exp_diff(float l, float top) {
    const float d = __fsub_rn(l, top), bb = __fsub_rn(d, l);
    const float r = __fsub_rn(__fsub_rn(l, __fsub_rn(d, bb)), __fadd_rn(top, bb));
    const float e = expf(d);
    return d < -200.0f ? 0.0f : fmaf(e, r, e);  // e is 0 there, and d may be infinite
}
// A score in fp32. Error: expf and log1pf are within 2 ulp (4 half ulps each), __fdividef
// within 2 ulp, the additions and the root half an ulp, so sigmoid and sqrt(softplus) are
// within 9 half ulps. Softmax divides by a sum of E terms exp(l - top). A term's exponent d is
// off by |d| half ulps, __expf by 4 + 2.4 |d|; weighted by the terms themselves the mean of |d|
// is at most ln E <= 7, and the chains are at most 37 additions long: the sum is within 4 + 3.4 *
// 7 + 37 = 65 half ulps, the score within 6 + 65 + 4 = 75.
template <int KIND>
__device__ __forceinline__ float score_f32(float l, float top, float sum) {
    if (KIND == CLB_SCORE_SIGMOID) return __fdividef(1.0f, 1.0f + expf(-l));
    if (KIND == CLB_SCORE_SOFTMAX) return __fdividef(exp_diff(l, top), sum);
    // far below, e^l and then the logarithm are no normal numbers long before their root e^(l/2) is (off by e^l / 4)
    return l < -20.0f ? expf(0.5f * l) : sqrtf(fmaxf(l, 0.0f) + log1pf(expf(-fabsf(l))));
}
// The same for the ranks' comparison alone, where what counts is the error in units of the row's
// largest score s(top) (u: half ulps), and a third of the instructions:
// - sigmoid: e = __expf(-l) is within 4 + 2.4 |l| u, s = 1 / (1 + e) within (1 - s) (4 + 2.4 |l|) + 5;
//   s |l| is at most 0.28 for l >= top >= -1.3, where s(top) >= 0.21, and else at most s(top) |top|:
//   within (13 + 2.4 max(0, -top)) u s(top).
// - sqrt(log(1 + e^l)), from log1p(e) = 2 atanh(z), z = e / (2 + e) <= 1/3, whose series to z^13 leaves
//   (1/9)^7 / 15: for l < 0 the logarithm is within 4 + 2.4 |l| + 9 u, its root within half of that and
//   2; s |l| is at most 0.72, s(-2) = 0.356: within (13 + 1.2 max(0, -top)) u s(top); l > 0 adds less.
// - softmax: the sum's own terms, each within e^d (4 + 3.4 |d|) u <= 5.3 u, times 1 / sum (2 u) and
//   rounded, over a sum within 65 u: within 74 u / sum.
// A score that is flushed to 0 is below 2^-63.
template <int KIND>
__device__ __forceinline__ float score_rough(float l) {
    if (KIND == CLB_SCORE_SIGMOID) return __fdividef(1.0f, 1.0f + __expf(-l));
    const float e = __expf(-fabsf(l)), z = __fdividef(e, 2.0f + e), t = z * z;
    float p = fmaf(t, 1.0f / 13.0f, 1.0f / 11.0f);
    p = fmaf(p, t, 1.0f / 9.0f);
    p = fmaf(p, t, 1.0f / 7.0f);
    p = fmaf(p, t, 1.0f / 5.0f);
    p = fmaf(p, t, 1.0f / 3.0f);
    p = fmaf(p, t, 1.0f);
    p = fmaf(z + z, p, fmaxf(l, 0.0f));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(p) : "f"(p));
    return p;
}
template <int KIND>
__device__ __noinline__ float score_exact(double l, double top, double sum) {
    if (KIND == CLB_SCORE_SIGMOID) return (float)(1.0 / (1.0 + exp(-l)));
    if (KIND == CLB_SCORE_SOFTMAX) return (float)(exp(l - top) / sum);
    return (float)sqrt(fmax(l, 0.0) + log1p(exp(-fabs(l))));
}
__device__ __noinline__ double exp_exact(float l, float top) { return exp((double)l - (double)top); }
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// One warp per token, expert e = 32 i + lane in the lane's i-th register (-inf behind the last).
// SCORED: the ranks or the groups' values need scores. A token's 1.5 KB of logits are read
// once; what bounds it is the latency of one warp's chain for few tokens and the issue slots
// for many (590 warp instructions a token in the last of these cases), so candidates for the picks are
// cut down by the lanes' maxima and ranked by counting instead of k passes over the row. Measured on a
// B200 (device time): 1 x 384, sigmoid and bias, k 6: 2.8 us; 61 x 384 in 8 groups: 3.5 us; 2048 x
// 384, sqrt-softplus and bias: 5.9 us (7.0 with expf, log1pf and a rounded root for the ranks);
// 16383 x 256 softmax, k 8: 11.6 us (1.5 TB/s). One pick after the other with all scores in double
// took 9.9, 15, 19 and 45 us. The form for more than 512 experts spills up to 224 bytes a thread, that for
// 384 up to 60: 2048 tokens, sigmoid and bias, 512 experts 5.6 us, 544 and 1024 10 us.
template <int NPL, int KIND, bool SCORED>
__global__ void __launch_bounds__(32 * kRouteWarps, NPL <= 12 ? 6 : NPL <= 16 ? 5 : 3) k_route_experts(const RouteArgs a) {
    __shared__ unsigned long long cand_s[kRouteWarps][32];                         // key, ~id
    __shared__ float vals_s[SCORED ? kRouteWarps : 1][SCORED ? NPL * 32 : 1];  // scores, then with their bias
    ops_wait();  // without letting the next kernel in early: its CTAs in this one's free slots made 2048 tokens 9.4 us, not 7.8
    const unsigned all = 0xffffffffu;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (t >= a.tokens) return;
    const int64_t row = t * a.ld;
    int* ids = a.ids + t * a.k;
    float* w = a.w + t * a.k;

    float l[NPL], b[NPL];
    {
        uint32_t raw[NPL];
        if (a.type == CLB_F32) {
            const uint32_t* p = static_cast<const uint32_t*>(a.logits) + row;
#pragma unroll
            for (int i = 0; i < NPL; ++i) raw[i] = p[min(32 * i + lane, a.E - 1)];
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row;
#pragma unroll
            for (int i = 0; i < NPL; ++i) raw[i] = p[min(32 * i + lane, a.E - 1)];
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) b[i] = 0.0f;
        if (a.bias)
#pragma unroll
            for (int i = 0; i < NPL; ++i) b[i] = a.bias[min(32 * i + lane, a.E - 1)];
        if (a.type == CLB_F32) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) l[i] = __uint_as_float(raw[i]);
        } else if (a.type == CLB_BF16) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) l[i] = __uint_as_float(raw[i] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) l[i] = __half2float(__ushort_as_half((uint16_t)raw[i]));
        }
    }
    float top = l[0], most = b[0];
#pragma unroll
    for (int i = 1; i < NPL; ++i) top = max_nan(top, l[i]), most = max_nan(most, b[i]);
    if (!__all_sync(all, top < INFINITY && most < INFINITY)) {
        if (lane == 0 && a.status) atomicExch(a.status, 1);
        if (lane < a.k) {
            ids[lane] = lane;
            w[lane] = __int_as_float(0x7fffffff);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        if (32 * i + lane >= a.E) l[i] = -INFINITY;
    float sum = 1.0f;
    if (KIND == CLB_SCORE_SOFTMAX || SCORED) top = fmaxf(warp_max(top), -FLT_MAX);
    if (KIND == CLB_SCORE_SOFTMAX) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float e = __expf(l[i] - top);
            sum += e;
            if (SCORED) vals_s[warp][32 * i + lane] = e;
        }
        sum = ops_warp_sum(sum);
    }
    // the largest error of a rough score, and of the scores below the normal numbers (from logits of -200 on
    // all are, so that -top enters as 200 at most: 2.5 times the lowest fp32 would be infinite, and off not a number)
    float off = 0.0f;
    if (SCORED && KIND == CLB_SCORE_SOFTMAX) off = fmaf(96.0f * kHalfUlp, __fdividef(1.0f, fmaxf(sum, 1.0f)), 1e-18f);
    else if (SCORED) off = fmaf(fmaf(fminf(fmaxf(-top, 0.0f), 200.0f), 2.5f, 16.0f) * kHalfUlp, score_rough<KIND>(top), 1e-18f);

    uint32_t mine = 0;      // lane j: the key and id of the j-th largest rank
    int id = 0;
    float lj = 0.0f, s;     // lane j < k: logit and score of its pick
    int exact = 0;
    auto exact_sum = [&] {
        double d = KIND == CLB_SCORE_SOFTMAX ? 0.0 : 1.0;
        if (KIND == CLB_SCORE_SOFTMAX) {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (l[i] > -INFINITY) d += exp_exact(l[i], top);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(all, d, o);
        }
        return d;
    };
#pragma unroll 1
    for (;;) {
        uint32_t key[NPL];
        if (SCORED) {
            if (!exact) {
                if (KIND != CLB_SCORE_SOFTMAX)
#pragma unroll
                    for (int i = 0; i < NPL; ++i) vals_s[warp][32 * i + lane] = score_rough<KIND>(l[i]);
            } else {  // rare: nothing kept in registers for it
                const double dsum = exact_sum();
#pragma unroll 1
                for (int e = lane; e < a.E; e += 32)
                    vals_s[warp][e] = score_exact<KIND>(ops_load(a.logits, a.type, row + e), top, dsum);
            }
        }
        const float by = KIND != CLB_SCORE_SOFTMAX || exact ? 1.0f : __fdividef(1.0f, sum);
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int e = 32 * i + lane;
            float v = l[i];
            if (SCORED) {
                // without a bias b is 0
                const float sc = __fadd_rn(KIND == CLB_SCORE_SOFTMAX ? __fmul_rn(vals_s[warp][e], by) : vals_s[warp][e], b[i]);
                const bool there = l[i] > -INFINITY && b[i] > -INFINITY;
                v = !there ? -INFINITY : a.bias ? sc : l[i];
                if (a.groups > 1) vals_s[warp][e] = there ? sc : -INFINITY;
            }
            key[i] = rank_key(v);
        }
        bool unsure = false;
        if (a.groups > 1) {
            // 2^log_lanes lanes find the two best of a group
            const int L = 1 << a.log_lanes, g = lane >> a.log_lanes;
            const bool mine_too = g < a.groups;
            float v1 = -INFINITY, v2 = -INFINITY;
            __syncwarp();
            if (mine_too) {
#pragma unroll 4
                for (int i = lane & (L - 1); i < a.per; i += L) {
                    const float v = SCORED ? vals_s[warp][g * a.per + i] : ops_load(a.logits, a.type, row + g * a.per + i);
                    v2 = fmaxf(v2, fminf(v1, v));
                    v1 = fmaxf(v1, v);
                }
            }
            __syncwarp();
            for (int o = 1; o < L; o <<= 1) {
                const float o1 = __shfl_xor_sync(all, v1, o), o2 = __shfl_xor_sync(all, v2, o);
                v2 = fmaxf(fmaxf(v2, o2), fminf(v1, o1));
                v1 = fmaxf(v1, o1);
            }
            // a group's place is the number of groups in front of it
            const float second = a.pair && v2 > -INFINITY ? v2 : 0.0f, value = __fadd_rn(v1, second);
            const uint32_t gkey = rank_key(value);
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < a.groups; ++j) {
                const uint32_t other = __shfl_sync(all, gkey, j << a.log_lanes);
                place += other > gkey || (other == gkey && j < g);
            }
            const bool keep = mine_too && place < a.top_groups;
            const unsigned kept = __ballot_sync(all, keep);
            if (SCORED && !exact) {
                // A value's error: 2 off of two scores, a rounding of each rank on both sides (of the rank's own size: the
                // two may cancel), the sum's and the bound's own: 5 u (|v1| + |second|). Other experts may be the two best
                // by exact ranks, but a rank and its error grow together, so the bound holds for whoever is.
                const float err = fmaf(6.0f * kHalfUlp, fabsf(v1), fmaf(6.0f * kHalfUlp, fabsf(second), 2.0f * off));
                const uint32_t last = __reduce_min_sync(all, keep ? rank_key(value - err) : 0xffffffffu);
                const uint32_t next = __reduce_max_sync(all, mine_too && !keep && value > -INFINITY ? rank_key(value + err) : 0u);
                unsure = next > kKeyNegInf && last <= next;
            }
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const int e = 32 * i + lane, ge = min((int)(((float)e + 0.5f) * a.per_inv), a.groups - 1);
                if (!((kept >> (ge << a.log_lanes)) & 1u)) key[i] = kKeyNegInf;
            }
        }
        // The k + 1 largest keys. The (k + 1)-th largest of the lanes' maxima is a lower bound of
        // them: the few keys from there on are collected, one to a lane, and ranked by counting.
        const int want = min(a.k + 1, a.E);
        uint32_t cur = key[0];
#pragma unroll
        for (int i = 1; i < NPL; ++i) cur = max(cur, key[i]);
        uint32_t bound = 0;
        for (int i = 0; i < want; ++i) {
            bound = __reduce_max_sync(all, cur);
            if (cur == bound) cur = 0;
        }
        // the keys from `from` on (the ids of equal keys ascending) into shared memory; their number
        auto collect = [&](uint32_t from) {
            int at = 0;
#pragma unroll
            for (int i = 0; i < NPL; ++i) at += key[i] >= from;
            const int own = at;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int before = __shfl_up_sync(all, at, o);
                if (lane >= o) at += before;
            }
            const int n = __shfl_sync(all, at, 31);
            at -= own;
            if (n <= 32)
#pragma unroll
                for (int i = 0; i < NPL; ++i)
                    if (key[i] >= from) cand_s[warp][at++] = (unsigned long long)key[i] << 32 | (uint32_t)~(32 * i + lane);
            __syncwarp();
            return n;
        };
        // lane j < n brings candidate j and takes the j-th largest
        float bj = 0.0f;
        auto order = [&](unsigned long long c, int n) {
            int place = 0;
            for (int j = 0; j < n; ++j) place += cand_s[warp][j] > c;
            __syncwarp();
            if (lane < n) cand_s[warp][place] = c;
            __syncwarp();
            c = lane < n ? cand_s[warp][lane] : 0ull;
            mine = (uint32_t)(c >> 32), id = (int)~(uint32_t)c;
            __syncwarp();
        };
        const int n = collect(max(bound, 1u));
        if (n <= 32) {
            order(cand_s[warp][lane], n);
        } else {  // many equal keys: one pick at a time
            uint32_t left[NPL];
#pragma unroll
            for (int i = 0; i < NPL; ++i) left[i] = key[i];
            for (int j = 0; j < want; ++j) {
                uint32_t best = 0, at = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < NPL; ++i)
                    if (left[i] > best) best = left[i], at = (uint32_t)(32 * i + lane);
                const uint32_t m = __reduce_max_sync(all, best);
                const uint32_t e = __reduce_min_sync(all, best == m ? at : 0xffffffffu);
#pragma unroll
                for (int i = 0; i < NPL; ++i)
                    if ((uint32_t)(32 * i + lane) == e) left[i] = 0;
                if (lane == j) mine = m, id = (int)e;
            }
        }
        auto pick_inputs = [&] {  // of lane j's pick; without scores the key is the logit
            if (!SCORED) {
                lj = key_value(mine);
            } else if (lane < want && mine) {  // after the second order there may be no (k + 1)-th
                lj = ops_load(a.logits, a.type, row + id);
                if (a.bias) bj = a.bias[id];
            }
        };
        pick_inputs();
        if (!SCORED || exact) break;
        if (__any_sync(all, unsure)) {  // of the groups
            exact = 1;
            continue;
        }
        if (!a.bias) break;
        // do the picks stand? Two experts of one logit and one bias have one rank, exactly
        const uint32_t nkey = __shfl_down_sync(all, mine, 1);
        const float nl = __shfl_down_sync(all, lj, 1), nb = __shfl_down_sync(all, bj, 1);
        const float v = key_value(mine), nv = key_value(nkey);
        if (lane + 1 < want && nkey != kKeyNegInf && !(lj == nl && bj == nb))
            unsure = !(v - nv > 2.0f * (off + kHalfUlp * (fabsf(v) + fabsf(nv))));
        // Where the last pick and the place behind it are such a pair, the best of the others decides (groups that
        // do not stay may be among them). From memory (64 x 384 bf16 with biases of 0: 4.1 us for 3.0): out of the registers it
        // took 3.3, but 0.1 us from every row without such a pair.
        const int cut = a.k - 1;
        if (__any_sync(all, lane == cut && cut + 1 < want && nkey != kKeyNegInf && lj == nl && bj == nb)) {
            const uint32_t own = __shfl_sync(all, mine, cut);
            const float pl = __shfl_sync(all, lj, cut), pb = __shfl_sync(all, bj, cut);
            uint32_t rest = 0;
#pragma unroll 4
            for (int e = lane; e < a.E; e += 32) {
                const float le = ops_load(a.logits, a.type, row + e), be = a.bias[e];
                float r = vals_s[warp][e];
                if (a.groups == 1) r = __fadd_rn(KIND == CLB_SCORE_SOFTMAX ? __fmul_rn(r, by) : r, be);
                const uint32_t ke = rank_key(r);
                if (ke <= own && le > -INFINITY && be > -INFINITY && !(le == pl && be == pb)) rest = max(rest, ke);
            }
            rest = __reduce_max_sync(all, rest);
            const float pv = key_value(own), rv = key_value(rest);
            unsure |= rest > kKeyNegInf && !(pv - rv > 2.0f * (off + kHalfUlp * (fabsf(pv) + fabsf(rv))));
        }
        if (!__any_sync(all, unsure)) break;
        // whoever can be among the picks: an exact rank for each, a lane apiece
        const float least = __shfl_sync(all, v, a.k - 1), margin = 4.0f * (off + 2.0f * kHalfUlp * fabsf(least));
        const int close = !(least > -INFINITY) ? 33 : collect(rank_key(least - margin));
        if (close > 32 || close < a.k) {  // the k picks are among them by construction
            exact = 1;
            continue;
        }
        unsigned long long c = lane < close ? cand_s[warp][lane] : 0ull;
        const double dsum = exact_sum();
        if (lane < close && (uint32_t)(c >> 32) != kKeyNegInf) {
            const int e = (int)~(uint32_t)c;
            const float se = score_exact<KIND>(ops_load(a.logits, a.type, row + e), top, dsum);
            c = (unsigned long long)rank_key(__fadd_rn(se, a.bias[e])) << 32 | (uint32_t)c;
            cand_s[warp][lane] = c;
        }
        __syncwarp();
        order(c, close);
        pick_inputs();
        break;
    }
    s = lane < a.k && mine != kKeyNegInf ? score_f32<KIND>(lj, top, sum) : 0.0f;
    if (a.renorm) {
        float total = 0.0f;
        for (int i = 0; i < a.k; ++i) total = __fadd_rn(total, __shfl_sync(all, s, i));
        s = __fdiv_rn(s, __fadd_rn(total, 1e-20f));
    }
    if (lane < a.k) {
        ids[lane] = id;
        w[lane] = __fmul_rn(s, a.scale);
    }
}

template <int KIND, bool SCORED>
void (*route_kernel(int per_lane))(RouteArgs) {
    return per_lane <= 4    ? k_route_experts<4, KIND, SCORED>
           : per_lane <= 8  ? k_route_experts<8, KIND, SCORED>
           : per_lane <= 12 ? k_route_experts<12, KIND, SCORED>
           : per_lane <= 16 ? k_route_experts<16, KIND, SCORED>
                            : k_route_experts<32, KIND, SCORED>;
}
template <bool SCORED>
void (*route_kernel(int kind, int per_lane))(RouteArgs) {
    return kind == CLB_SCORE_SIGMOID   ? route_kernel<CLB_SCORE_SIGMOID, SCORED>(per_lane)
           : kind == CLB_SCORE_SOFTMAX ? route_kernel<CLB_SCORE_SOFTMAX, SCORED>(per_lane)
                                       : route_kernel<CLB_SCORE_SQRT_SOFTPLUS, SCORED>(per_lane);
}

}  // namespace
}  // namespace clb

extern "C" int32_t clb_route_experts_device(const clb_route_config_v1* cfg, const void* d_logits, int64_t ld,
                                            const float* d_bias, int32_t tokens, int32_t* d_ids, float* d_w,
                                            int32_t* d_status, void* stream, clb_error_v1* err) {
    return guarded(err, [&] {
        require(cfg != nullptr, CLB_E_INVALID, "null routing config");
        const clb_route_config_v1 c = *cfg;
        require(c.n_experts >= 1 && c.n_experts <= clb::kRouteMaxExperts, CLB_E_INVALID,
                "n_experts = %d, not in 1..%d", c.n_experts, clb::kRouteMaxExperts);
        require(c.score >= CLB_SCORE_SIGMOID && c.score <= CLB_SCORE_SQRT_SOFTPLUS, CLB_E_INVALID,
                "unknown routing score %d", c.score);
        require(c.n_groups >= 1 && c.n_groups <= clb::kRouteMaxGroups && c.n_experts % c.n_groups == 0, CLB_E_INVALID,
                "n_groups = %d: not in 1..%d, or does not divide %d experts", c.n_groups, clb::kRouteMaxGroups,
                c.n_experts);
        require(c.top_groups >= 1 && c.top_groups <= c.n_groups, CLB_E_INVALID, "top_groups = %d of %d groups",
                c.top_groups, c.n_groups);
        require(c.n_groups == 1 || c.group_score == CLB_GROUP_MAX || c.group_score == CLB_GROUP_PAIR, CLB_E_INVALID,
                "unknown group score %d", c.group_score);
        require(c.k >= 1 && c.k <= clb::kRouteMaxPicks && c.k <= c.top_groups * (c.n_experts / c.n_groups),
                CLB_E_INVALID, "k = %d: not in 1..%d, or more than the kept groups' experts", c.k,
                clb::kRouteMaxPicks);
        require(c.renormalize == 0 || c.renormalize == 1, CLB_E_INVALID, "renormalize is 0 or 1");
        require(std::isfinite(c.scale) && c.scale >= 0, CLB_E_INVALID, "route scale must be finite and >= 0");
        require(clb::ops_float_type(c.logits_type), CLB_E_INVALID, "logits are fp32, bf16 or fp16");
        require(!c.reserved[0] && !c.reserved[1] && !c.reserved[2], CLB_E_INVALID, "reserved fields must be 0");
        require(tokens >= 0 && ld >= c.n_experts, CLB_E_INVALID, "invalid token count or row pitch");
        if (tokens == 0) return;
        require(d_logits && d_ids && d_w, CLB_E_INVALID, "null pointer argument");
        require(clb::ops_aligned(d_logits, clb::ops_type_bytes(c.logits_type)) && clb::ops_aligned(d_bias, 4) &&
                    clb::ops_aligned(d_ids, 4) && clb::ops_aligned(d_w, 4) && clb::ops_aligned(d_status, 4),
                CLB_E_INVALID, "misaligned pointer argument");
        const clb::OpsRows in[] = {clb::ops_rows("logits", d_logits, tokens, c.n_experts, ld, c.logits_type),
                                   clb::ops_rows("bias", d_bias, 1, c.n_experts, c.n_experts, CLB_F32)};
        const clb::OpsRows ids = clb::ops_rows("ids", d_ids, 1, (int64_t)tokens * c.k, 0, CLB_F32);
        const clb::OpsRows w = clb::ops_rows("weights", d_w, 1, (int64_t)tokens * c.k, 0, CLB_F32), to_w[] = {w};
        clb::ops_require_apart(ids, in);
        clb::ops_require_apart(w, in);
        clb::ops_require_apart(ids, to_w);
        // groups that all stay decide nothing (9972 x 88, 2 of 2 groups, sigmoid: 7.6 us, 12.1 with their values)
        const int groups = c.top_groups < c.n_groups ? c.n_groups : 1;
        clb::RouteArgs a{d_logits, d_bias, d_ids, d_w, d_status, ld, tokens, c.logits_type, c.n_experts, c.k, groups,
                         c.top_groups, c.group_score == CLB_GROUP_PAIR, c.renormalize, c.n_experts / groups, 0, c.scale,
                         (float)groups / (float)c.n_experts};
        while ((2 * a.groups) << a.log_lanes <= 32) ++a.log_lanes;
        const bool scored = d_bias || (a.groups > 1 && a.pair);
        const int per_lane = (c.n_experts + 31) / 32;
        cuda_check(clb::ops_launch(scored ? clb::route_kernel<true>(c.score, per_lane) : clb::route_kernel<false>(c.score, per_lane),
                                   (unsigned)(((int64_t)tokens + clb::kRouteWarps - 1) / clb::kRouteWarps), 32 * clb::kRouteWarps, 0,
                                   static_cast<cudaStream_t>(stream), a),
                   "routing");
    });
}
