// The residual step between two blocks: RMSNorm after the block, gate, scaled residual sum,
// RMSNorm before the next block, in one pass over the rows.
//
// One CTA per row holds the row in registers: y and h are read once, h' and x written once,
// so the kernel is bound by those bytes. The two sums of squares are fp32: per thread in
// element order, then over the warp and the CTA in a fixed tree.
#include <algorithm>
#include <cmath>

#include "clb_ops.cuh"

namespace clb {
namespace {

constexpr int kNormMaxDim = 32768;

struct NormArgs {
    const void *h, *y, *gate;
    const float *w_post, *w_pre;
    void *h_out, *x;
    int64_t ld_h, ld_y, ld_gate, ld_h_out, ld_x;
    int dim, h_type, y_type, gate_type, x_type, gate_kind, gate_sigmoid, post;
    float post_eps, pre_eps, residual_scale, block_scale, inv_dim;
};

// Sum over the CTA, the same bits in every thread. `part`: 32 floats, not those of the
// previous call.
__device__ __forceinline__ float cta_sum(float v, float* part) {
    v = ops_warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    return ops_warp_sum(lane < nw ? part[lane] : 0.0f);
}

// Eight values of a thread's chunk (coherent loads: h may be updated in place). VEC: 8 contiguous elements, 16-byte loads. Otherwise
// the elements are blockDim apart, so that a warp's scalar accesses stay contiguous.
template <bool VEC>
__device__ __forceinline__ void load8(const void* p, int type, int64_t base, int chunk, int dim, float (&v)[8]) {
    if (VEC) {
        load8_aligned(p, type, base + (int64_t)chunk * 8, v);
    } else {
        const int i = chunk / (int)blockDim.x, tid = chunk % (int)blockDim.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = (i * 8 + j) * (int)blockDim.x + tid;
            v[j] = e < dim ? ops_load(p, type, base + e) : 0.0f;
        }
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(void* p, int type, int64_t base, int chunk, int dim, const float (&v)[8]) {
    if (VEC) {
        const int64_t i = base + (int64_t)chunk * 8;
        if (type == CLB_F32) {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
            q[0] = make_float4(v[0], v[1], v[2], v[3]);
            q[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (type == CLB_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&b);
                } else {
                    const __half2 b = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&b);
                }
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        const int i = chunk / (int)blockDim.x, tid = chunk % (int)blockDim.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = (i * 8 + j) * (int)blockDim.x + tid;
            if (e < dim) ops_store(p, type, base + e, v[j]);
        }
    }
}

__device__ __forceinline__ float gate_value(float g, int sigmoid) {
    return sigmoid ? 1.0f / (1.0f + expf(-g)) : g;
}

// CH chunks of 8 values per thread.
template <int CH, bool VEC>
__global__ void __launch_bounds__(1024) k_block_norm(const NormArgs a) {
    __shared__ float part[2][32];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int chunks = VEC ? a.dim >> 3 : 0x7fffffff;  // scalar chunks mask element by element
    float v[CH][8], y[CH][8];
    if (a.y) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (tid + c * nt < chunks) load8<VEC>(a.y, a.y_type, row * a.ld_y, tid + c * nt, a.dim, y[c]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) y[c][j] = 0.0f;
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (tid + c * nt < chunks) load8<VEC>(a.h, a.h_type, row * a.ld_h, tid + c * nt, a.dim, v[c]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
    }
    if (a.y) {
        float inv = 1.0f;
        if (a.post) {
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(y[c][j], y[c][j], ss);
            inv = 1.0f / sqrtf(cta_sum(ss, part[0]) * a.inv_dim + a.post_eps);
        }
        float gt = 1.0f;
        if (a.gate_kind == CLB_GATE_TOKEN) gt = gate_value(ops_load(a.gate, a.gate_type, row), a.gate_sigmoid);
        const float f = a.block_scale * gt * inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int ch = tid + c * nt;
            if (ch < chunks) {
                if (a.post && a.w_post) {
                    float w[8];
                    load8<VEC>(a.w_post, CLB_F32, 0, ch, a.dim, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[c][j] *= w[j];
                }
                if (a.gate_kind == CLB_GATE_CHANNEL || a.gate_kind == CLB_GATE_FULL) {
                    float g[8];
                    load8<VEC>(a.gate, a.gate_type, a.gate_kind == CLB_GATE_FULL ? row * a.ld_gate : 0, ch, a.dim, g);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[c][j] *= gate_value(g[j], a.gate_sigmoid);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = fmaf(f, y[c][j], a.residual_scale * v[c][j]);
                store8<VEC>(a.h_out, a.h_type, row * a.ld_h_out, ch, a.dim, v[c]);
            }
        }
    }
    if (a.x) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(v[c][j], v[c][j], ss);
        const float inv = 1.0f / sqrtf(cta_sum(ss, part[1]) * a.inv_dim + a.pre_eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int ch = tid + c * nt;
            if (ch < chunks) {
                float w[8];
                if (a.w_pre) {
                    load8<VEC>(a.w_pre, CLB_F32, 0, ch, a.dim, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] *= v[c][j] * inv;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = v[c][j] * inv;
                }
                store8<VEC>(a.x, a.x_type, row * a.ld_x, ch, a.dim, w);
            }
        }
    }
}

}  // namespace
}  // namespace clb

extern "C" int32_t clb_block_norm_device(const clb_block_norm_config_v1* cfg, int32_t tokens, const void* d_h,
                                         const void* d_y, const void* d_gate, const float* d_w_post,
                                         const float* d_w_pre, void* d_h_out, void* d_x, void* stream,
                                         clb_error_v1* err) {
    return guarded(err, [&] {
        require(cfg != nullptr, CLB_E_INVALID, "null block norm config");
        const clb_block_norm_config_v1 c = *cfg;
        require(c.dim >= 1 && c.dim <= clb::kNormMaxDim, CLB_E_INVALID, "dim = %d, not in 1..%d", c.dim,
                clb::kNormMaxDim);
        require(clb::ops_float_type(c.h_type) && clb::ops_float_type(c.y_type) && clb::ops_float_type(c.gate_type) &&
                    clb::ops_float_type(c.x_type),
                CLB_E_INVALID, "tensors are fp32, bf16 or fp16");
        require((c.post == 0 || c.post == 1) && (c.gate_sigmoid == 0 || c.gate_sigmoid == 1) &&
                    c.gate >= CLB_GATE_NONE && c.gate <= CLB_GATE_FULL,
                CLB_E_INVALID, "invalid norm or gate kind");
        require(std::isfinite(c.post_eps) && c.post_eps > 0 && std::isfinite(c.pre_eps) && c.pre_eps > 0, CLB_E_INVALID,
                "eps must be finite and > 0");
        require(std::isfinite(c.residual_scale) && std::isfinite(c.block_scale), CLB_E_INVALID,
                "residual and block scale must be finite");
        for (int i = 0; i < 4; ++i) require(!c.reserved[i], CLB_E_INVALID, "reserved fields must be 0");
        require(tokens >= 0, CLB_E_INVALID, "negative token count");
        if (tokens == 0) return;
        require(d_h && (d_y || d_x), CLB_E_INVALID, "null pointer argument: h and one of y and x are needed");
        require((d_y != nullptr) == (d_h_out != nullptr), CLB_E_INVALID, "h_out goes with y");
        require(d_y || (!d_gate && !d_w_post), CLB_E_INVALID, "a gate or w_post without y");
        require(!d_y || (d_gate != nullptr) == (c.gate != CLB_GATE_NONE), CLB_E_INVALID,
                "the gate pointer goes with the gate kind");
        require(!d_w_post || c.post, CLB_E_INVALID, "w_post without the norm after the block");
        require(!d_w_pre || d_x, CLB_E_INVALID, "w_pre without x");
        struct Tensor { const void* p; int type; int64_t ld; const char* name; };
        const bool full = d_gate && c.gate == CLB_GATE_FULL;
        const Tensor rows[] = {{d_h, c.h_type, c.ld_h, "h"}, {d_y, c.y_type, c.ld_y, "y"},
                               {full ? d_gate : nullptr, c.gate_type, c.ld_gate, "gate"},
                               {d_h_out, c.h_type, c.ld_h_out, "h_out"}, {d_x, c.x_type, c.ld_x, "x"}};
        const Tensor vecs[] = {{full ? nullptr : d_gate, c.gate_type, 0, "gate"}, {d_w_post, CLB_F32, 0, "w_post"},
                               {d_w_pre, CLB_F32, 0, "w_pre"}};
        bool vec = c.dim % 8 == 0;
        for (const Tensor& t : rows) {
            if (!t.p) continue;
            const size_t b = clb::ops_type_bytes(t.type);
            require(t.ld >= c.dim && t.ld <= (int64_t)1 << 40, CLB_E_INVALID, "row pitch of %s below dim", t.name);
            require(clb::ops_aligned(t.p, b), CLB_E_INVALID, "%s is misaligned", t.name);
            vec = vec && clb::ops_aligned(t.p, 16) && t.ld * b % 16 == 0;
        }
        for (const Tensor& t : vecs) {
            if (!t.p) continue;
            require(clb::ops_aligned(t.p, clb::ops_type_bytes(t.type)), CLB_E_INVALID, "%s is misaligned", t.name);
            // a gate for each token is read one number at a time
            if (t.p != d_gate || c.gate == CLB_GATE_CHANNEL) vec = vec && clb::ops_aligned(t.p, 16);
        }
        // an output over an input: only h_out in h's place, row by row
        const Tensor outs[] = {rows[3], rows[4]};
        for (int o = 0; o < 2; ++o) {
            if (!outs[o].p) continue;
            const char* lo = static_cast<const char*>(outs[o].p);
            const char* hi = lo + ((tokens - 1) * outs[o].ld + c.dim) * clb::ops_type_bytes(outs[o].type);
            for (int i = 0; i < 5; ++i) {
                const Tensor& t = rows[i];
                if (!t.p || i == 3 + o) continue;
                if (i == 0 && o == 0 && t.p == outs[o].p && t.ld == outs[o].ld) continue;
                const char* l = static_cast<const char*>(t.p);
                const char* h = l + ((tokens - 1) * t.ld + c.dim) * clb::ops_type_bytes(t.type);
                // rows of one wider buffer may interleave: same pitch in bytes, disjoint columns
                const int64_t pitch = t.ld * clb::ops_type_bytes(t.type);
                bool apart = hi <= l || h <= lo;
                if (!apart && pitch == outs[o].ld * clb::ops_type_bytes(outs[o].type)) {
                    const int64_t wo = (int64_t)c.dim * clb::ops_type_bytes(outs[o].type);
                    const int64_t wt = (int64_t)c.dim * clb::ops_type_bytes(t.type);
                    const int64_t d = (((lo - l) % pitch) + pitch) % pitch;  // column of the output after t's start
                    apart = d >= wt && d + wo <= pitch;
                }
                require(apart, CLB_E_INVALID, "%s overlaps %s", outs[o].name, t.name);
            }
        }
        clb::NormArgs a{};
        a.h = d_h, a.y = d_y, a.gate = d_gate, a.w_post = d_w_post, a.w_pre = d_w_pre, a.h_out = d_h_out, a.x = d_x;
        a.ld_h = c.ld_h, a.ld_y = c.ld_y, a.ld_gate = c.ld_gate, a.ld_h_out = c.ld_h_out, a.ld_x = c.ld_x;
        a.dim = c.dim, a.h_type = c.h_type, a.y_type = c.y_type, a.gate_type = c.gate_type, a.x_type = c.x_type;
        a.gate_kind = d_gate ? c.gate : CLB_GATE_NONE, a.gate_sigmoid = c.gate_sigmoid, a.post = c.post;
        a.post_eps = c.post_eps, a.pre_eps = c.pre_eps, a.residual_scale = c.residual_scale;
        a.block_scale = c.block_scale, a.inv_dim = 1.0f / (float)c.dim;
        const int units = (c.dim + 7) / 8;
        const int ch = units <= 1024 ? 1 : units <= 2048 ? 2 : 4;
        const int threads = std::max(32, ((units + ch - 1) / ch + 31) / 32 * 32);
        void (*kernel)(clb::NormArgs) = vec ? (ch == 1   ? clb::k_block_norm<1, true>
                                               : ch == 2 ? clb::k_block_norm<2, true>
                                                         : clb::k_block_norm<4, true>)
                                            : (ch == 1   ? clb::k_block_norm<1, false>
                                               : ch == 2 ? clb::k_block_norm<2, false>
                                                         : clb::k_block_norm<4, false>);
        cuda_check(clb::ops_launch(kernel, (unsigned)tokens, threads, 0, static_cast<cudaStream_t>(stream), a),
                   "block norm");
    });
}
