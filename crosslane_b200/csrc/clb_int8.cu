// Matrix product in 8-bit integers with a scale for each token and output channel:
//   out[t][n] = x_scale[t] * w_scale[n] * sum_k q[t][k] * w[n][k] (+ bias[n]),
// the sum exact in 32-bit integers, and the quantisation of rows that makes q and w.
//
// Quantisation. scale = fl(max |x| / 127); q is the integer nearest to x / scale, decided on
// the exact quotient: an fp32 quotient can round onto the border between two integers. With
// q0 the rounded fp32 quotient, r = x - q0 * scale is exact in one fused multiply-add (both
// terms are multiples of half an ulp of scale and |r| < scale), so comparing 2 |r| with
// scale settles the neighbour. Rows whose scale is below 2^-100 are first lifted by 2^100
// (exact, the quotients stay), so that 1 / scale and the remainders are normal numbers.
#include <algorithm>
#include <cmath>

#include "clb_ops.cuh"

namespace clb {
namespace {

constexpr int kInt8MaxK = 131072;  // 127 * 127 * k stays below 2^31
constexpr int kErrInt8Wait = 3;

__device__ __forceinline__ int quant_one(float x, float scale, float inv) {
    float q = rintf(x * inv);
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    const float r = fmaf(-q, scale, x), two = r + r;
    if (two > scale || (two == scale && ((int)q & 1))) q += 1.0f;
    else if (two < -scale || (two == -scale && ((int)q & 1))) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// One CTA per row.
__global__ void __launch_bounds__(256) k_int8_quantize(const void* __restrict__ x, int type, int64_t ld_x, int k,
                                                       int8_t* __restrict__ q, int64_t ld_q, int kpad,
                                                       float* __restrict__ scale) {
    __shared__ float part[8];
    __shared__ int bad_s;
    const int64_t row = blockIdx.x;
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    float m = 0.0f;
    bool bad = false;
    for (int i = threadIdx.x; i < k; i += 256) {
        const float v = fabsf(ops_load(x, type, row * ld_x + i));
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    if (bad) bad_s = 1;
    __syncthreads();
    m = part[0];
    for (int i = 1; i < 8; ++i) m = fmaxf(m, part[i]);
    const float s = __fdiv_rn(m, 127.0f);
    const bool zero = bad_s || !(s > 0.0f);
    const float lift = s < 0x1p-100f ? 0x1p100f : 1.0f, ls = s * lift, inv = zero ? 0.0f : __fdiv_rn(1.0f, ls);
    for (int i = threadIdx.x; i < kpad; i += 256)
        q[row * ld_q + i] = zero || i >= k ? 0 : (int8_t)quant_one(ops_load(x, type, row * ld_x + i) * lift, ls, inv);
    if (threadIdx.x == 0) scale[row] = bad_s ? __int_as_float(0x7fffffff) : s;
}

struct Int8Args {
    const int8_t *w, *q;
    const float *w_scale, *q_scale, *bias;
    void* out;
    int64_t ld_w, ld_q, ld_out;
    int tokens, n, k, out_type;
};

__device__ __forceinline__ float int8_value(int acc, float xs, float ws, float bias, bool has_bias) {
    const float v = __fmul_rn(__fmul_rn((float)acc, xs), ws);
    return has_bias ? __fadd_rn(v, bias) : v;
}

// One warp per weight row and up to 8 tokens.
__global__ void __launch_bounds__(256) k_int8_dot(const Int8Args a) {
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (n >= a.n) return;
    const int t0 = blockIdx.y * 8, nt = min(8, a.tokens - t0);
    const int8_t* w = a.w + n * a.ld_w;
    int acc[8] = {};
    for (int p = lane; p < a.k >> 4; p += 32) {
        const int4 wv = reinterpret_cast<const int4*>(w)[p];
        for (int t = 0; t < nt; ++t) {
            const int4 v = reinterpret_cast<const int4*>(a.q + (t0 + t) * a.ld_q)[p];
            acc[t] = __dp4a(wv.x, v.x, __dp4a(wv.y, v.y, __dp4a(wv.z, v.z, __dp4a(wv.w, v.w, acc[t]))));
        }
    }
    for (int i = (a.k & ~15) + lane; i < a.k; i += 32)
        for (int t = 0; t < nt; ++t) acc[t] += (int)w[i] * (int)a.q[(t0 + t) * a.ld_q + i];
    for (int t = 0; t < nt; ++t) {
        const int s = __reduce_add_sync(0xffffffffu, acc[t]);
        if (lane == 0)
            ops_store(a.out, a.out_type, (t0 + t) * a.ld_out + n,
                      int8_value(s, a.q_scale[t0 + t], a.w_scale[n], a.bias ? a.bias[n] : 0.0f, a.bias != nullptr));
    }
}

int64_t round16(int64_t v) { return (v + 15) & ~(int64_t)15; }

}  // namespace
}  // namespace clb

extern "C" int32_t clb_int8_quantize_device(int32_t type, const void* d_x, int64_t ld_x, int32_t rows, int32_t k,
                                            int8_t* d_q, int64_t ld_q, float* d_scale, void* stream,
                                            clb_error_v1* err) {
    return guarded(err, [&] {
        require(clb::ops_float_type(type), CLB_E_INVALID, "x is fp32, bf16 or fp16");
        require(k >= 1 && k <= clb::kInt8MaxK, CLB_E_INVALID, "k = %d, not in 1..%d", k, clb::kInt8MaxK);
        require(rows >= 0 && ld_x >= k && ld_q >= k && ld_q % 16 == 0, CLB_E_INVALID,
                "invalid row count or pitch (ld_q is a multiple of 16)");
        if (rows == 0) return;
        require(d_x && d_q && d_scale, CLB_E_INVALID, "null pointer argument");
        require(clb::ops_aligned(d_x, clb::ops_type_bytes(type)) && clb::ops_aligned(d_q, 16) &&
                    clb::ops_aligned(d_scale, 4),
                CLB_E_INVALID, "misaligned pointer argument (q is 16-byte aligned)");
        cuda_check(clb::ops_launch(clb::k_int8_quantize, (unsigned)rows, 256, 0, static_cast<cudaStream_t>(stream), d_x,
                                   type, ld_x, k, d_q, ld_q, k, d_scale),
                   "int8 quantise");
    });
}

extern "C" uint64_t clb_int8_linear_workspace_bytes(int32_t tokens, int32_t k) {
    if (tokens < 0 || k < 1 || k > clb::kInt8MaxK) return 0;
    return (uint64_t)tokens * clb::round16(k) + clb::round16((int64_t)tokens * 4) + 16;
}

extern "C" int32_t clb_int8_linear_device(const clb_int8_linear_config_v1* cfg, const int8_t* d_w,
                                          const float* d_w_scale, const float* d_bias, int32_t tokens,
                                          const void* d_x, const float* d_x_scale, void* d_out, void* d_ws,
                                          uint64_t ws_bytes, int32_t* d_status, void* stream, clb_error_v1* err) {
    return guarded(err, [&] {
        require(cfg != nullptr, CLB_E_INVALID, "null int8 linear config");
        const clb_int8_linear_config_v1 c = *cfg;
        const bool ready = c.x_type == CLB_I8;
        require(c.n >= 1 && c.k >= 1 && c.k <= clb::kInt8MaxK, CLB_E_INVALID, "n >= 1 and k in 1..%d", clb::kInt8MaxK);
        require((ready || clb::ops_float_type(c.x_type)) && clb::ops_float_type(c.out_type), CLB_E_INVALID,
                "x is fp32, bf16, fp16 or int8; out is fp32, bf16 or fp16");
        require(c.ld_w >= c.k && c.ld_w % 16 == 0, CLB_E_INVALID, "ld_w is a multiple of 16, at least k");
        require(c.ld_x >= c.k && (!ready || c.ld_x % 16 == 0), CLB_E_INVALID,
                "ld_x is at least k (a multiple of 16 for int8)");
        require(c.ld_out >= c.n, CLB_E_INVALID, "ld_out below n");
        for (int i = 0; i < 4; ++i) require(!c.reserved[i], CLB_E_INVALID, "reserved fields must be 0");
        require(tokens >= 0, CLB_E_INVALID, "negative token count");
        if (tokens == 0) return;
        require(d_w && d_w_scale && d_x && d_out, CLB_E_INVALID, "null pointer argument");
        require(ready == (d_x_scale != nullptr), CLB_E_INVALID, "x_scale goes with int8 x");
        require(clb::ops_aligned(d_w, 16) && clb::ops_aligned(d_w_scale, 4) && clb::ops_aligned(d_bias, 4) &&
                    clb::ops_aligned(d_x, ready ? 16 : clb::ops_type_bytes(c.x_type)) &&
                    clb::ops_aligned(d_x_scale, 4) && clb::ops_aligned(d_out, clb::ops_type_bytes(c.out_type)) &&
                    clb::ops_aligned(d_ws, 16) && clb::ops_aligned(d_status, 4),
                CLB_E_INVALID, "misaligned pointer argument");
        require(ready || (d_ws && ws_bytes >= clb_int8_linear_workspace_bytes(tokens, c.k)), CLB_E_INVALID,
                "workspace below clb_int8_linear_workspace_bytes");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        clb::Int8Args a{d_w, nullptr, d_w_scale, nullptr, d_bias, d_out, c.ld_w, 0, c.ld_out, tokens, c.n, c.k,
                        c.out_type};
        if (ready) {
            a.q = static_cast<const int8_t*>(d_x);
            a.q_scale = d_x_scale;
            a.ld_q = c.ld_x;
        } else {
            a.ld_q = clb::round16(c.k);
            float* scale = reinterpret_cast<float*>(static_cast<int8_t*>(d_ws) + tokens * a.ld_q);
            a.q = static_cast<const int8_t*>(d_ws);
            a.q_scale = scale;
            cuda_check(clb::ops_launch(clb::k_int8_quantize, (unsigned)tokens, 256, 0, s, d_x, c.x_type, c.ld_x, c.k,
                                       static_cast<int8_t*>(d_ws), a.ld_q, (int)a.ld_q, scale),
                       "int8 quantise");
        }
        cuda_check(clb::ops_launch(clb::k_int8_dot, dim3((unsigned)((c.n + 7) / 8), (unsigned)((tokens + 7) / 8)), 256,
                                   0, s, a),
                   "int8 product");
    });
}
