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
    int lanes_per_group;  // power of two, groups * lanes_per_group <= 32
    float scale, per_inv;  // per_inv: groups / E
};

// Order-preserving map of a float to unsigned (-0 as +0); 0 is below every key.
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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
// within 9 half ulps; softmax divides by a sum of E terms whose chains are at most 37
// additions long: within 6 + 6 + 37 + 4 half ulps.
template <int KIND>
__device__ __forceinline__ float score_f32(float l, float top, float sum) {
    if (KIND == CLB_SCORE_SIGMOID) return __fdividef(1.0f, 1.0f + expf(-l));
    if (KIND == CLB_SCORE_SOFTMAX) return __fdividef(exp_diff(l, top), sum);
    return sqrtf(fmaxf(l, 0.0f) + log1pf(expf(-fabsf(l))));
}
template <int KIND>
__device__ __noinline__ float score_exact(double l, double top, double sum) {
    if (KIND == CLB_SCORE_SIGMOID) return (float)(1.0 / (1.0 + exp(-l)));
    if (KIND == CLB_SCORE_SOFTMAX) return (float)(exp(l - top) / sum);
    return (float)sqrt(fmax(l, 0.0) + log1p(exp(-fabs(l))));
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// One warp per token, expert e = 32 i + lane in the lane's i-th register. SCORED: the ranks or the
// groups' values need scores. Bound by latency and instructions (a token's 1.5 KB of logits
// are read once).
template <int NPL, int KIND, bool SCORED>
__global__ void __launch_bounds__(32 * kRouteWarps, NPL <= 12 ? 6 : NPL <= 16 ? 5 : 3) k_route_experts(const RouteArgs a) {
    __shared__ uint4 cand_s[kRouteWarps][32];                                      // key, id, logit, bias
    __shared__ float vals_s[SCORED ? kRouteWarps : 1][SCORED ? NPL * 32 : 1];  // scores, then with their bias
    const unsigned all = 0xffffffffu;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * kRouteWarps + warp;
    if (t >= a.tokens) return;
    const int64_t row = (int64_t)t * a.ld;
    int* ids = a.ids + (int64_t)t * a.k;
    float* w = a.w + (int64_t)t * a.k;

    float l[NPL], b[NPL];
    {
        uint32_t raw[NPL];
        if (a.type == CLB_F32) {
            const uint32_t* p = static_cast<const uint32_t*>(a.logits) + row;
#pragma unroll
            for (int i = 0; i < NPL; ++i) raw[i] = __ldg(p + min(32 * i + lane, a.E - 1));
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row;
#pragma unroll
            for (int i = 0; i < NPL; ++i) raw[i] = __ldg(p + min(32 * i + lane, a.E - 1));
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) b[i] = 0.0f;
        if (a.bias)
#pragma unroll
            for (int i = 0; i < NPL; ++i) b[i] = __ldg(a.bias + min(32 * i + lane, a.E - 1));
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
    bool fine = true;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        fine = fine && l[i] < INFINITY && b[i] < INFINITY;
        top = fmaxf(top, l[i]);
    }
    if (!__all_sync(all, fine)) {
        if (lane == 0 && a.status) atomicExch(a.status, 1);
        if (lane < a.k) {
            ids[lane] = lane;
            w[lane] = __int_as_float(0x7fffffff);
        }
        return;
    }
    float sum = 1.0f;
    if (KIND == CLB_SCORE_SOFTMAX || SCORED) top = warp_max(top);
    if (KIND == CLB_SCORE_SOFTMAX) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (32 * i + lane < a.E && l[i] > -INFINITY) sum += exp_diff(l[i], top);
        sum = ops_warp_sum(sum);
    }
    // the largest error of a score (s rises with l), and of the scores below the normal numbers
    const float off = !SCORED ? 0.0f
                              : fmaf(KIND == CLB_SCORE_SOFTMAX ? 64.0f * kHalfUlp : 16.0f * kHalfUlp,
                                     KIND == CLB_SCORE_SQRT_SOFTPLUS ? score_f32<KIND>(top, 0.0f, 1.0f) : 1.0f, 1e-18f);

    uint32_t mine = 0;      // lane j: the key and id of the j-th largest rank
    int id = 0;
    float lj = 0.0f, s;     // lane j < k: logit and score of its pick
    int exact = 0;
#pragma unroll 1
    for (;;) {
        uint32_t key[NPL];
        if (SCORED) {
            if (!exact) {
#pragma unroll
                for (int i = 0; i < NPL; ++i) vals_s[warp][32 * i + lane] = score_f32<KIND>(l[i], top, sum);
            } else {  // rare: nothing kept in registers for it
                double dsum = 1.0;
                if (KIND == CLB_SCORE_SOFTMAX) {
                    dsum = 0.0;
#pragma unroll 1
                    for (int e = lane; e < a.E; e += 32) {
                        const float le = ops_load(a.logits, a.type, row + e);
                        if (le > -INFINITY) dsum += exp((double)le - (double)top);
                    }
                    for (int o = 16; o > 0; o >>= 1) dsum += __shfl_xor_sync(all, dsum, o);
                }
#pragma unroll 1
                for (int e = lane; e < a.E; e += 32)
                    vals_s[warp][e] = score_exact<KIND>(ops_load(a.logits, a.type, row + e), top, dsum);
            }
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int e = 32 * i + lane;
            float v = l[i];
            if (SCORED) {
                const float sc = __fadd_rn(vals_s[warp][e], b[i]);  // without a bias b is 0
                const bool there = l[i] > -INFINITY && b[i] > -INFINITY;
                v = !there ? -INFINITY : a.bias ? sc : l[i];
                if (a.groups > 1) vals_s[warp][e] = there ? sc : -INFINITY;
            }
            key[i] = e < a.E ? rank_key(v) : 0u;
        }
        bool unsure = false;
        if (a.groups > 1) {
            // lanes_per_group lanes find the two best of a group
            const int per = a.E / a.groups, L = a.lanes_per_group, g = lane / L;
            float v1 = -INFINITY, v2 = -INFINITY;
            __syncwarp();
            if (g < a.groups)
                for (int i = lane % L; i < per; i += L) {
                    const float v = SCORED ? vals_s[warp][g * per + i] : ops_load(a.logits, a.type, row + g * per + i);
                    v2 = fmaxf(v2, fminf(v1, v));
                    v1 = fmaxf(v1, v);
                }
            __syncwarp();
            for (int o = 1; o < L; o <<= 1) {
                const float o1 = __shfl_xor_sync(all, v1, o), o2 = __shfl_xor_sync(all, v2, o);
                v2 = fmaxf(fmaxf(v2, o2), fminf(v1, o1));
                v1 = fmaxf(v1, o1);
            }
            const float value = a.pair && v2 > -INFINITY ? __fadd_rn(v1, v2) : v1;
            uint32_t gkey = g < a.groups && lane % L == 0 ? rank_key(value) : 0u;
            uint32_t kept = 0, last = 0;
            for (int i = 0; i < a.top_groups; ++i) {
                last = __reduce_max_sync(all, gkey);
                const int at = __ffs(__ballot_sync(all, gkey == last)) - 1;
                kept |= 1u << (at / L);
                if (lane == at) gkey = 0;
            }
            if (SCORED && !exact && a.top_groups < a.groups) {
                // a value's error: of two scores, of their ranks' roundings and of the sum's
                const uint32_t next = __reduce_max_sync(all, gkey);
                const float lo = key_value(last), hi = key_value(next);
                unsure = next != kKeyNegInf && !(lo - hi > 4.0f * (off + 2.0f * kHalfUlp * (fabsf(lo) + fabsf(hi))));
            }
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const int e = 32 * i + lane, ge = (int)(((float)e + 0.5f) * a.per_inv);
                if (e < a.E && !((kept >> ge) & 1u)) key[i] = kKeyNegInf;
            }
        }
        // The k + 1 largest keys. The (k + 1)-th largest of the lanes' maxima is a lower bound of
        // them: the few keys from there on are collected, one to a lane, and ranked by counting.
        const int want = min(a.k + 1, a.E);
        uint32_t cur = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) cur = max(cur, key[i]);
        uint32_t bound = 0;
        for (int i = 0; i < want; ++i) {
            bound = __reduce_max_sync(all, cur);
            if (cur == bound) cur = 0;
        }
        // the keys from `from` on into shared memory, in the order of the ids; their number
        auto collect = [&](uint32_t from) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const unsigned m = __ballot_sync(all, key[i] >= from);
                if (m) {
                    const int at = n + __popc(m & ((1u << lane) - 1u));
                    if (key[i] >= from && at < 32)
                        cand_s[warp][at] =
                            make_uint4(key[i], (uint32_t)(32 * i + lane), __float_as_uint(l[i]), __float_as_uint(b[i]));
                    n += __popc(m);
                }
            }
            __syncwarp();
            return n;
        };
        // lane j < n brings a candidate, collected as its j-th, and takes the j-th largest
        float bj = 0.0f;
        auto order = [&](uint4 c, int n) {
            int place = 0;
            for (int j = 0; j < n; ++j) {
                const uint32_t ok = cand_s[warp][j].x;
                place += ok > c.x || (ok == c.x && j < lane);
            }
            __syncwarp();
            if (lane < n) cand_s[warp][place] = c;
            __syncwarp();
            c = cand_s[warp][lane];
            mine = c.x, id = (int)c.y, lj = __uint_as_float(c.z), bj = __uint_as_float(c.w);
            __syncwarp();
        };
        const int n = collect(max(bound, 1u));  // keys of 0 are no experts
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
            if (lane < want) {
                lj = ops_load(a.logits, a.type, row + id);
                if (a.bias) bj = a.bias[id];
            }
        }
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
        if (!__any_sync(all, unsure)) break;
        // whoever can be among the picks: an exact rank for each, a lane apiece
        const float least = __shfl_sync(all, v, a.k - 1), margin = 4.0f * (off + 2.0f * kHalfUlp * fabsf(least));
        const int close = KIND == CLB_SCORE_SOFTMAX || !(least > -INFINITY) ? 33 : collect(rank_key(least - margin));
        if (close > 32) {
            exact = 1;
            continue;
        }
        uint4 c = cand_s[warp][lane];
        if (lane < close && c.x != kKeyNegInf)
            c.x = rank_key(__fadd_rn(score_exact<KIND>(__uint_as_float(c.z), 0.0, 1.0), __uint_as_float(c.w)));
        if (lane < close) cand_s[warp][lane].x = c.x;
        __syncwarp();
        order(c, close);
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
        clb::RouteArgs a{d_logits, d_bias, d_ids, d_w, d_status, ld, tokens, c.logits_type, c.n_experts, c.k, c.n_groups,
                         c.top_groups, c.group_score == CLB_GROUP_PAIR, c.renormalize, 1, c.scale,
                         (float)c.n_groups / (float)c.n_experts};
        while (2 * a.lanes_per_group * a.groups <= 32) a.lanes_per_group *= 2;
        const bool scored = d_bias || (a.groups > 1 && a.pair);
        const int per_lane = (c.n_experts + 31) / 32;
        cuda_check(clb::ops_launch(scored ? clb::route_kernel<true>(c.score, per_lane) : clb::route_kernel<false>(c.score, per_lane),
                                   (unsigned)((tokens + clb::kRouteWarps - 1) / clb::kRouteWarps), 32 * clb::kRouteWarps, 0,
                                   static_cast<cudaStream_t>(stream), a),
                   "routing");
    });
}
