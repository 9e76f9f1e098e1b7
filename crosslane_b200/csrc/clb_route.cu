// Routing to experts for models whose routing is neither of clb_route_device's modes: scores
// of three kinds, a bias for balance, groups of experts, top-k, renormalised weights.
//
// Ranks are compared as fp32 values that are the same on every machine: a score is evaluated
// in double and rounded once (the correctly rounded float, up to double's own last bits), the
// bias is added in fp32, and ties go to the lower id. Without a bias the rank is the logit,
// since every score rises with it, and only the picks' scores are evaluated.
#include <cmath>

#include "clb_ops.cuh"

namespace clb {
namespace {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxPicks = 16;
constexpr int kRouteMaxGroups = 32;
constexpr int kRouteWarps = 4;
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // rank_key(-inf): an expert that is not available

struct RouteArgs {
    const void* logits;
    const float* bias;
    int* ids;
    float* w;
    int* status;
    int64_t ld;
    int tokens, type, E, k, score, groups, top_groups, pair, renorm;
    float scale;
};

// Order-preserving map of a float to unsigned (-0 as +0); 0 is below every key.
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ double score_of(int kind, double l, double top, double sum) {
    if (kind == CLB_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-l));
    if (kind == CLB_SCORE_SOFTMAX) return exp(l - top) / sum;
    return sqrt(fmax(l, 0.0) + log1p(exp(-fabs(l))));
}

// One warp per token; the row's keys and scores in shared memory.
__global__ void __launch_bounds__(32 * kRouteWarps) k_route_experts(const RouteArgs a) {
    extern __shared__ float route_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * kRouteWarps + warp;
    if (t >= a.tokens) return;
    uint32_t* key = reinterpret_cast<uint32_t*>(route_smem) + (size_t)warp * 2 * a.E;
    float* sc = reinterpret_cast<float*>(key + a.E);
    const int64_t row = (int64_t)t * a.ld;
    const unsigned all = 0xffffffffu;

    bool bad = false;
    float top = -INFINITY;
    for (int e = lane; e < a.E; e += 32) {
        const float l = ops_load(a.logits, a.type, row + e);
        const float b = a.bias ? __ldg(a.bias + e) : 0.0f;
        bad |= !(l < INFINITY) || !(b < INFINITY);
        top = fmaxf(top, l);
    }
    if (__any_sync(all, bad)) {
        if (lane == 0 && a.status) atomicExch(a.status, 1);
        for (int i = lane; i < a.k; i += 32) {
            a.ids[(int64_t)t * a.k + i] = i;
            a.w[(int64_t)t * a.k + i] = __int_as_float(0x7fffffff);
        }
        return;
    }
    double sum = 0.0;
    if (a.score == CLB_SCORE_SOFTMAX) {
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(all, top, o));
        for (int e = lane; e < a.E; e += 32) {
            const float l = ops_load(a.logits, a.type, row + e);
            if (l > -INFINITY) sum += exp((double)l - (double)top);
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(all, sum, o);
    }
    const bool pair = a.groups > 1 && a.pair;
    for (int e = lane; e < a.E; e += 32) {
        const float l = ops_load(a.logits, a.type, row + e);
        const float b = a.bias ? __ldg(a.bias + e) : 0.0f;
        uint32_t u = kKeyNegInf;
        float s = 0.0f;
        if (l > -INFINITY && b > -INFINITY) {
            if (a.bias || pair) s = (float)score_of(a.score, l, top, sum);
            u = rank_key(a.bias ? __fadd_rn(s, b) : l);
        }
        key[e] = u;
        sc[e] = a.bias ? __fadd_rn(s, b) : s;  // what a pair of a group adds up
    }
    __syncwarp();
    if (a.groups > 1) {
        const int per = a.E / a.groups;
        uint32_t gkey = 0;
        if (lane < a.groups) {
            uint32_t best = kKeyNegInf;
            float v1 = -INFINITY, v2 = -INFINITY;
            for (int i = 0; i < per; ++i) {
                const uint32_t u = key[lane * per + i];
                best = max(best, u);
                if (u != kKeyNegInf) {
                    const float v = sc[lane * per + i];
                    v2 = fmaxf(v2, fminf(v1, v));
                    v1 = fmaxf(v1, v);
                }
            }
            gkey = !a.pair ? best : rank_key(v2 > -INFINITY ? __fadd_rn(v1, v2) : v1);
        }
        uint32_t kept = 0;
        for (int i = 0; i < a.top_groups; ++i) {
            const uint32_t m = __reduce_max_sync(all, gkey);
            const int g = __ffs(__ballot_sync(all, gkey == m)) - 1;
            kept |= 1u << g;
            if (lane == g) gkey = 0;
        }
        for (int e = lane; e < a.E; e += 32)
            if (!((kept >> (e / per)) & 1u)) key[e] = kKeyNegInf;
        __syncwarp();
    }
    float mine = 0.0f;
    int id = 0;
    float total = 0.0f;
    for (int i = 0; i < a.k; ++i) {
        uint32_t best = 0;
        int be = 0;
        for (int e = lane; e < a.E; e += 32)
            if (key[e] > best) best = key[e], be = e;
        const uint32_t m = __reduce_max_sync(all, best);
        const int e = (int)__reduce_min_sync(all, best == m ? (unsigned)be : 0xffffffffu);
        if (e % 32 == lane) key[e] = 0;
        float s = 0.0f;
        if (m != kKeyNegInf) s = (float)score_of(a.score, ops_load(a.logits, a.type, row + e), top, sum);
        total = __fadd_rn(total, s);
        if (lane == i) mine = s, id = e;
        __syncwarp();
    }
    if (lane < a.k) {
        if (a.renorm) mine = __fdiv_rn(mine, __fadd_rn(total, 1e-20f));
        a.ids[(int64_t)t * a.k + lane] = id;
        a.w[(int64_t)t * a.k + lane] = __fmul_rn(mine, a.scale);
    }
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
        clb::RouteArgs a{d_logits, d_bias, d_ids, d_w, d_status, ld, tokens, c.logits_type, c.n_experts, c.k, c.score,
                         c.n_groups, c.top_groups, c.group_score == CLB_GROUP_PAIR, c.renormalize, c.scale};
        cuda_check(clb::ops_launch(clb::k_route_experts, (unsigned)((tokens + clb::kRouteWarps - 1) / clb::kRouteWarps),
                                   32 * clb::kRouteWarps, (size_t)clb::kRouteWarps * 2 * c.n_experts * 4,
                                   static_cast<cudaStream_t>(stream), a),
                   "routing");
    });
}
