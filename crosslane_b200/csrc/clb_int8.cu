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
#include "clb_tc.cuh"

namespace clb {
namespace {

constexpr int kInt8MaxK = 131072;  // 127 * 128 * k stays below 2^31
constexpr int kInt8MaxRows = 1 << 30;  // weight rows, tokens: their tiles are counted in int
constexpr int kErrInt8Wait = 3;

// The exactly rounded quotient; `inv` the fp32 reciprocal of scale.
__device__ __forceinline__ int quant_exact(float x, float scale, float inv) {
    float q = rintf(x * inv);
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    const float r = fmaf(-q, scale, x), two = r + r;
    if (two > scale || (two == scale && ((int)q & 1))) q += 1.0f;
    else if (two < -scale || (two == -scale && ((int)q & 1))) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// What a row's values are divided by. tiny: the row is lifted by 2^100 first, and its largest
// quotient may pass 127 (scale is a subnormal number).
struct RowScale {
    float scale, inv;
    bool zero, tiny;
};
__device__ __forceinline__ RowScale row_scale(float m, float* stored) {
    const float s = __fdiv_rn(m, 127.0f);
    RowScale r;
    r.zero = !(m < INFINITY) || !(s > 0.0f);  // m: largest |x|, NaN or infinite if the row holds such a value
    r.tiny = s < 0x1p-100f;
    r.scale = r.tiny ? s * 0x1p100f : s;
    r.inv = r.zero ? 0.0f : __fdiv_rn(1.0f, r.scale);
    *stored = m < INFINITY ? s : __int_as_float(0x7fffffff);
    return r;
}
// Eight quotients as bytes, of rows whose scale is a subnormal number (out of line).
__device__ __noinline__ uint2 quant8_exact(float v0, float v1, float v2, float v3, float v4, float v5, float v6, float v7,
                                           float scale, float inv, float lift) {
    const float v[8] = {v0, v1, v2, v3, v4, v5, v6, v7};
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = (uint32_t)quant_exact(v[j] * lift, scale, inv) & 0xffu;
    return make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
}
// The low byte of the result is the integer nearest to x / scale, for a quotient t = x * inv that is
// within 127 * 2^-22.4 = 2.4e-5 of it and was rounded by adding 1.5 * 2^23 (f): where t lies so
// close to a border, the exact remainder moves the integer by one if it has to be.
__device__ __forceinline__ uint32_t quant_settle(float x, float f, float scale) {
    const float r = fmaf(-(f - 12582912.0f), scale, x), two = fabsf(r + r);
    const uint32_t q = __float_as_uint(f);
    const bool move = two > scale || (two == scale && (q & 1u));
    return !move ? q : r > 0.0f ? q + 1u : q - 1u;
}
constexpr float kQuantSure = 0.49997f;  // a rounding to a distance below this stands

// Eight quotients as bytes. Values of 16 bits hit the borders exactly every few hundred times, so
// that path is short too; tiny rows take the general form.
__device__ __forceinline__ uint2 quant8(const float (&v)[8], const RowScale& r) {
    constexpr float kRound = 12582912.0f;
    const F2 inv = f2(r.inv, r.inv), round = f2(kRound, kRound), minus = f2(-1.0f, -1.0f);
    float f[8], off = 0.0f;
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const F2 t = f2_mul(f2(v[j], v[j + 1]), inv), u = f2_add(t, round);
        const float2 d = f2_floats(f2_add(t, f2_fma(u, minus, round)));  // from the rounded quotient
        const float2 uf = f2_floats(u);
        f[j] = uf.x, f[j + 1] = uf.y;
        q[j] = __float_as_uint(uf.x), q[j + 1] = __float_as_uint(uf.y);
        off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
    }
    if (off > kQuantSure)
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = quant_settle(v[j], f[j], r.scale);
    uint2 b = make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                         __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
    if (r.zero) b = make_uint2(0u, 0u);
    else if (r.tiny) b = quant8_exact(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], r.scale, r.inv, 0x1p100f);
    return b;
}
__device__ __forceinline__ int8_t quant1(float v, const RowScale& r) {
    if (r.zero) return 0;
    if (r.tiny) return (int8_t)quant_exact(v * 0x1p100f, r.scale, r.inv);
    const float t = v * r.inv, f = t + 12582912.0f;
    return (int8_t)(fabsf(t - (f - 12582912.0f)) > kQuantSure ? quant_settle(v, f, r.scale) : __float_as_uint(f));
}
// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float warp_max_nan(float m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

struct QuantArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t ld_x, ld_q;
    int k, limit;  // columns of x; columns of q that are written (zeros behind k)
};
__device__ __forceinline__ const void* row_at(const void* x, int type, int64_t element) {
    return static_cast<const char*>(x) + element * (type == CLB_F32 ? 4 : 2);
}
// The largest magnitude of a row from the threads' own, the same in every thread.
__device__ __forceinline__ float cta_max_nan(float m, float* part) {
    m = warp_max_nan(m);
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    return warp_max_nan(lane < (int)(blockDim.x >> 5) ? part[lane] : 0.0f);
}
// The largest magnitude of eight aligned values and m (NaN if there is one); two at a time in 16 bits.
template <int TYPE>
__device__ __forceinline__ float max8_nan(const Raw8& r, float m) {
    if (TYPE == CLB_F32) {
        float v[8];
        raw8_floats(r, TYPE, true, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
        return m;
    }
    if (TYPE == CLB_BF16) {
        auto part = [](const uint32_t& w) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)); };
        const __nv_bfloat162 x = __hmax2_nan(__hmax2_nan(part(r.a.x), part(r.a.y)), __hmax2_nan(part(r.a.z), part(r.a.w)));
        return max_nan(m, max_nan(__low2float(x), __high2float(x)));
    }
    auto part = [](const uint32_t& w) { return __habs2(*reinterpret_cast<const __half2*>(&w)); };
    const __half2 x = __hmax2_nan(__hmax2_nan(part(r.a.x), part(r.a.y)), __hmax2_nan(part(r.a.z), part(r.a.w)));
    return max_nan(m, max_nan(__low2float(x), __high2float(x)));
}

// A CTA per row, CH chunks of 8 values a thread in registers; or (CH = 0) rows too long for that,
// read twice. Rows that start anywhere (not ALIGNED) come through shared memory. The columns behind
// the last whole chunk are single values of the first threads. fp32 rows are bound by their bytes: 4096 x 7168
// 23.5 us (6.2 TB/s). 16-bit rows are not: bf16 21.7 us, fp16 18.3 us (4.1 and 4.8 TB/s); bf16 has 17
// instructions a value, 13.8 us of issue slots, and what its warps wait for most are the loads. In rows
// that start anywhere fp32 takes 32 and bf16 29 us; 64 x 5120 bf16 2.0 us.
template <int CH, int TYPE, bool ALIGNED>
__global__ void __launch_bounds__(1024) k_int8_quantize(const QuantArgs a) {
    __shared__ float part[32];
    ops_begin();
    const int tid = threadIdx.x, nt = blockDim.x, chunks = a.k >> 3, last = 8 * chunks + tid;
    const void* x = row_at(a.x, TYPE, (int64_t)blockIdx.x * a.ld_x);
    int8_t* q = a.q + (int64_t)blockIdx.x * a.ld_q;
    extern __shared__ uint4 row_smem[];
    const uint32_t smem = (uint32_t)__cvta_generic_to_shared(row_smem), off = (uint32_t)reinterpret_cast<uintptr_t>(x) & 15u;
    Raw8 raw[CH ? CH : 1];
    float v[8], m = 0.0f;
    if (!ALIGNED) {
        row_to_smem(smem, x, (uint32_t)a.k * (TYPE == CLB_F32 ? 4u : 2u), TYPE);
        row_landed();
    }
    if (CH)
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = tid + i * nt;
            if (ALIGNED) raw[i] = raw8_aligned(x, TYPE, 8 * (int64_t)c, c < chunks);
            else raw[i] = c < chunks ? raw8_smem(smem, off, TYPE, c) : Raw8{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        }
    const float tail = last < a.k ? ops_load(x, TYPE, last) : 0.0f;
    if (CH) {
#pragma unroll
        for (int i = 0; i < CH; ++i) m = max8_nan<TYPE>(raw[i], m);
    } else {
#pragma unroll 4
        for (int c = tid; c < chunks; c += nt) m = max8_nan<TYPE>(raw8_aligned(x, TYPE, 8 * (int64_t)c, true), m);
    }
    float stored;
    const RowScale r = row_scale(cta_max_nan(max_nan(m, fabsf(tail)), part), &stored);
    if (CH) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (tid + i * nt < chunks) {
                raw8_floats(raw[i], TYPE, true, v);
                *reinterpret_cast<uint2*>(q + 8 * (tid + i * nt)) = quant8(v, r);
            }
    } else {
#pragma unroll 2
        for (int c = tid; c < chunks; c += nt) {
            raw8_floats(raw8_aligned(x, TYPE, 8 * (int64_t)c, true), TYPE, true, v);
            *reinterpret_cast<uint2*>(q + 8 * c) = quant8(v, r);
        }
    }
    if (last < a.limit) q[last] = last < a.k ? quant1(tail, r) : 0;  // limit - 8 chunks < 24 values
    if (tid == 0) a.scale[blockIdx.x] = stored;
}

// Many short rows: a warp each, so that no CTA is started and joined for a row. CH chunks of 8 values a
// lane; in rows that start anywhere (not ALIGNED) the values are 32 apart.
template <int CH, int TYPE, bool ALIGNED>
__global__ void __launch_bounds__(256) k_int8_quantize_short(const QuantArgs a, int rows) {
    ops_begin();
    const int lane = threadIdx.x & 31, chunks = a.k >> 3;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const void* x = row_at(a.x, TYPE, row * a.ld_x);
    int8_t* q = a.q + row * a.ld_q;
    Raw8 raw[CH];
    float v[8], m = 0.0f, stored;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = lane + 32 * i;
        raw[i] = ALIGNED ? raw8_aligned(x, TYPE, 8 * (int64_t)c, c < chunks) : raw8_strided(x, TYPE, 256 * i + lane, 32, a.k);
    }
    const int last = 8 * chunks + lane;
    const float tail = ALIGNED && last < a.k ? ops_load(x, TYPE, last) : 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (ALIGNED) {
            m = max8_nan<TYPE>(raw[i], m);
        } else {
            raw8_floats(raw[i], TYPE, false, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
        }
    }
    const RowScale r = row_scale(warp_max_nan(max_nan(m, fabsf(tail))), &stored);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        raw8_floats(raw[i], TYPE, ALIGNED, v);
        if (ALIGNED) {
            if (lane + 32 * i < chunks) *reinterpret_cast<uint2*>(q + 8 * (lane + 32 * i)) = quant8(v, r);
        } else {
            const uint2 b = quant8(v, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = 256 * i + 32 * j + lane;
                if (e < a.limit) q[e] = (int8_t)((j < 4 ? b.x : b.y) >> (8 * (j & 3)));  // zeros behind k
            }
        }
    }
    if (ALIGNED && last < a.limit) q[last] = last < a.k ? quant1(tail, r) : 0;
    if (lane == 0) a.scale[row] = stored;
}

// Rows of any alignment too long for shared memory, value by value, read twice (the second time
// from L1 or L2).
template <int TYPE>
__global__ void __launch_bounds__(1024) k_int8_quantize_any(const QuantArgs a) {
    __shared__ float part[32];
    ops_begin();
    const int tid = threadIdx.x, nt = blockDim.x;
    const void* x = row_at(a.x, TYPE, (int64_t)blockIdx.x * a.ld_x);
    int8_t* q = a.q + (int64_t)blockIdx.x * a.ld_q;
    float m = 0.0f;
#pragma unroll 8
    for (int i = tid; i < a.k; i += nt) m = max_nan(m, fabsf(ops_load(x, TYPE, i)));
    float stored;
    const RowScale r = row_scale(cta_max_nan(m, part), &stored);
#pragma unroll 4
    for (int i = tid; i < a.limit; i += nt) q[i] = i < a.k ? quant1(ops_load(x, TYPE, i), r) : 0;
    if (tid == 0) a.scale[blockIdx.x] = stored;
}

template <int TYPE>
void (*quantize_kernel(int ch, bool vec))(QuantArgs) {
    return !vec ? (ch == 0   ? k_int8_quantize_any<TYPE>
                   : ch == 1 ? k_int8_quantize<1, TYPE, false>
                             : k_int8_quantize<4, TYPE, false>)
                : (ch == 0   ? k_int8_quantize<0, TYPE, true>
                   : ch == 1 ? k_int8_quantize<1, TYPE, true>
                             : k_int8_quantize<4, TYPE, true>);
}

template <int TYPE>
void (*short_kernel(int ch, bool vec))(QuantArgs, int) {
    return vec ? (ch == 1   ? k_int8_quantize_short<1, TYPE, true>
                  : ch == 2 ? k_int8_quantize_short<2, TYPE, true>
                            : k_int8_quantize_short<4, TYPE, true>)
               : (ch == 1 ? k_int8_quantize_short<1, TYPE, false> : k_int8_quantize_short<2, TYPE, false>);
}

// `limit`: columns written (k, or a pitch of a multiple of 16 whose rest is zeros).
cudaError_t launch_int8_quantize(const void* x, int type, int64_t ld_x, int rows, int k, int8_t* q, int64_t ld_q,
                                 int limit, float* scale, cudaStream_t s) {
    const QuantArgs a{x, q, scale, ld_x, ld_q, k, limit};
    const bool vec = ops_vec8(x, type, ld_x);
    const int units = (limit + 7) / 8;
    // Measured, a CTA a row and a warp a row: 2000 x 256 bf16 2.4 and 1.9 us, 8192 x 512 fp32 9.0 and 3.8 us
    // (8192 CTAs take 9 us to start), 8192 x 1024 9.4 and 8.2, unaligned 12.1 and 11.7; 600 x 256 1.7
    // either way, 600 x 512 1.7 and 1.8, 600 x 1024 unaligned 2.3 and 3.2 us.
    if (units <= 32 || (units <= (vec ? 128 : 64) && rows >= 1500)) {
        const int ch = units <= 32 ? 1 : units <= 64 ? 2 : 4;
        void (*kernel)(QuantArgs, int) = type == CLB_F32    ? short_kernel<CLB_F32>(ch, vec)
                                         : type == CLB_BF16 ? short_kernel<CLB_BF16>(ch, vec)
                                                            : short_kernel<CLB_F16>(ch, vec);
        return ops_launch(kernel, (unsigned)(((int64_t)rows + 7) / 8), 256, 0, s, a, rows);
    }
    // few rows: as many threads as the row has chunks, for the latency; many: 4 chunks a thread, so that
    // several rows of an SM overlap their loads and stores
    const size_t staged = vec ? 0 : (size_t)k * ops_type_bytes(type) + 48;
    const bool whole = units <= 4096 && staged <= 47 * 1024;  // with the static shared memory, below 48 KB
    const int ch = !whole ? 0 : units > 1024 || (rows > 296 && units > 128) ? 4 : 1;
    const int per = ch ? ch : vec ? 128 : 8;
    const int threads = std::min(1024, std::max(32, ((units * (vec || ch ? 1 : 8) + per - 1) / per + 31) / 32 * 32));
    void (*kernel)(QuantArgs) = type == CLB_F32    ? quantize_kernel<CLB_F32>(ch, vec)
                                : type == CLB_BF16 ? quantize_kernel<CLB_BF16>(ch, vec)
                                                   : quantize_kernel<CLB_F16>(ch, vec);
    return ops_launch(kernel, (unsigned)rows, threads, ch ? staged : 0, s, a);
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

// ------------------------------------------------------------------------------
// Few tokens (TT >= tokens): row dots on dp4a. Bound by the weights' bytes, so there is one launch
// and the first weights are in flight before the tokens are quantised: every CTA does that
// by itself into shared memory (x comes from L2; floating x) or copies q (int8 x). A CTA has
// `rows` weight rows, cut into 2^log_segs pieces of K that its warps share out; a piece's sums
// are integers, added in shared memory in any order. Measured on a B200 (device time, weights
// in part from L2), fp32 x: 1 token, 7168 x 1536 4.4 us (2.5 TB/s), 7168 x 7168 7.8 us; 4 tokens,
// 512 x 1024 3.8 us, 7168 x 7168 13.8 us (5.7 and 16.3 us with one token quantised after the
// other). 8 tokens took 4.3 us for the tiles' 5.2 at 512 x 1024, but 8.9 for 7.5 at 4096 x 2304 and
// 24 for 13 at 7168 x 7168.
constexpr int kDotThreads = 1024;
constexpr int kDotAhead = 4;                 // 16-byte weight pieces of a lane's group, two groups in flight
constexpr int kDotSmem = 160 * 1024;         // largest tokens * pitch that is staged
constexpr int kDotMaxSums = 8192;            // rows * tokens of a CTA
constexpr int kDotSmemMax = kDotSmem + 4 * kDotMaxSums;

struct Int8Dot {
    Int8Args a;
    const void* x;      // floating x, or null: a.q and a.q_scale are given
    int64_t ld_x;
    int rows, log_segs, kpad;
};

// TYPE: of a floating x.
template <int TT, bool VEC, int TYPE>
__global__ void __launch_bounds__(kDotThreads, 1) k_int8_dot(const Int8Dot d) {
    extern __shared__ uint4 dot_smem[];
    __shared__ float part[kDotThreads / 32], scale_s[TT];
    ops_begin();
    const Int8Args& a = d.a;
    int8_t* qs = reinterpret_cast<int8_t*>(dot_smem);               // [TT][kpad]
    int* sums = reinterpret_cast<int*>(qs + (size_t)TT * d.kpad);   // [rows][TT]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = blockIdx.x * d.rows, nr = min(d.rows, a.n - r0);
    const int pieces = a.k >> 4, per = (pieces + (1 << d.log_segs) - 1) >> d.log_segs;
    // A warp's share: items (a row's piece of K) warp, warp + 32, ..., each in groups of 32 * kDotAhead
    // weight pieces. The next group is asked for before one is multiplied, the first before the
    // tokens are quantised.
    struct Place {
        int item, at, end;
        const int4* row;
    };
    const int items = nr << d.log_segs;
    auto start = [&](int item) {
        const int seg = item & ((1 << d.log_segs) - 1);
        return Place{item, seg * per, item < items ? min(pieces, (seg + 1) * per) : 0,
                     reinterpret_cast<const int4*>(a.w + (int64_t)(r0 + (item >> d.log_segs)) * a.ld_w)};
    };
    auto advance = [&](Place p) {
        p.at += 32 * kDotAhead;
        return p.at < p.end ? p : start(p.item + kDotThreads / 32);
    };
    auto fetch = [&](int4 (&w)[kDotAhead], const Place& p) {
#pragma unroll
        for (int u = 0; u < kDotAhead; ++u) {
            const int i = p.at + lane + 32 * u;
            w[u] = make_int4(0, 0, 0, 0);
            if (i < p.end) w[u] = p.row[i];
        }
    };
    Place here = start(warp);
    int4 next[kDotAhead];
    fetch(next, here);
    for (int i = tid; i < d.rows * TT; i += kDotThreads) sums[i] = 0;
    // a token's threads, one after the other in it
    constexpr int kGroup = kDotThreads / TT, kWarps = kGroup / 32;
    const int own = tid / kGroup, at = tid % kGroup;
    int8_t* q = qs + (size_t)own * d.kpad;
    if (d.x) {
        // whole chunks, and the columns behind them as single values (zeros behind k)
        const int whole = VEC ? a.k >> 3 : 0, last = 8 * whole + at;
        const void* x = row_at(d.x, TYPE, min(own, a.tokens - 1) * d.ld_x);
        float m = 0.0f, v[8];
#pragma unroll 4
        for (int c = at; c < whole; c += kGroup) m = max8_nan<TYPE>(raw8_aligned(x, TYPE, 8 * (int64_t)c, true), m);
#pragma unroll 4
        for (int i = last; i < a.k; i += kGroup) m = max_nan(m, fabsf(ops_load(x, TYPE, i)));
        m = warp_max_nan(m);
        if (lane == 0) part[warp] = m;
        __syncthreads();
        float stored;
        const RowScale r = row_scale(warp_max_nan(part[own * kWarps + (lane & (kWarps - 1))]), &stored);
        if (own < a.tokens) {
#pragma unroll 2
            for (int c = at; c < whole; c += kGroup) {
                raw8_floats(raw8_aligned(x, TYPE, 8 * (int64_t)c, true), TYPE, true, v);
                *reinterpret_cast<uint2*>(q + 8 * c) = quant8(v, r);
            }
#pragma unroll 2
            for (int i = last; i < d.kpad; i += kGroup) q[i] = i < a.k ? quant1(ops_load(x, TYPE, i), r) : 0;
            if (at == 0) scale_s[own] = stored;
        }
    } else if (own < a.tokens) {
        for (int p = at; p < pieces; p += kGroup) reinterpret_cast<int4*>(q)[p] = reinterpret_cast<const int4*>(a.q + own * a.ld_q)[p];
        for (int i = 16 * pieces + at; i < a.k; i += kGroup) q[i] = a.q[own * a.ld_q + i];
        if (at == 0) scale_s[own] = a.q_scale[own];
    }
    __syncthreads();
    int acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = 0;
    while (here.item < items) {
        int4 w[kDotAhead];
#pragma unroll
        for (int u = 0; u < kDotAhead; ++u) w[u] = next[u];
        const Place then = advance(here);
        fetch(next, then);
#pragma unroll
        for (int u = 0; u < kDotAhead; ++u) {
            if (here.at + 32 * u >= here.end) break;
            const int p = min(here.at + lane + 32 * u, pieces - 1);  // weights behind the end are zero
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int4 v = reinterpret_cast<const int4*>(qs + (size_t)t * d.kpad)[p];
                acc[t] = __dp4a(w[u].x, v.x, __dp4a(w[u].y, v.y, __dp4a(w[u].z, v.z, __dp4a(w[u].w, v.w, acc[t]))));
            }
        }
        if (then.item != here.item) {
            const int row = here.item >> d.log_segs;
            if ((~here.item & ((1 << d.log_segs) - 1)) == 0) {  // the columns behind the last whole piece
                const int i = 16 * pieces + lane;
                if (i < a.k) {
                    const int wv = a.w[(int64_t)(r0 + row) * a.ld_w + i];
#pragma unroll
                    for (int t = 0; t < TT; ++t)
                        if (t < a.tokens) acc[t] += wv * qs[(size_t)t * d.kpad + i];
                }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int sum = __reduce_add_sync(0xffffffffu, acc[t]);
                acc[t] = 0;
                if (lane == 0) {
                    if (d.log_segs == 0) sums[row * TT + t] = sum;
                    else atomicAdd(&sums[row * TT + t], sum);
                }
            }
        }
        here = then;
    }
    __syncthreads();
    for (int i = tid; i < nr * a.tokens; i += kDotThreads) {
        const int t = i / nr, r = i % nr, n = r0 + r;
        ops_store(a.out, a.out_type, t * a.ld_out + n,
                  int8_value(sums[r * TT + t], scale_s[t], a.w_scale[n], a.bias ? a.bias[n] : 0.0f, a.bias != nullptr));
    }
}

template <int TT, bool VEC>
void (*dot_kernel(int type))(Int8Dot) {
    return type == CLB_F32    ? k_int8_dot<TT, VEC, CLB_F32>
           : type == CLB_BF16 ? k_int8_dot<TT, VEC, CLB_BF16>
                              : k_int8_dot<TT, VEC, CLB_F16>;
}
void (*dot_kernel(int tt, bool vec, int type))(Int8Dot) {
    return vec ? (tt == 1 ? dot_kernel<1, true>(type) : tt == 2 ? dot_kernel<2, true>(type) : dot_kernel<4, true>(type))
               : (tt == 1 ? dot_kernel<1, false>(type) : tt == 2 ? dot_kernel<2, false>(type) : dot_kernel<4, false>(type));
}

// ------------------------------------------------------------------------------
// Tensor-core product: D[weight rows][nt tokens] in tensor memory (int32), A = weights and B =
// quantised tokens by TMA (128-byte rows of K, 128-byte swizzle), four tcgen05.mma kind::i8 of
// K = 32 per 128-byte block. Warps 0-7 are the epilogue (a lane is a weight row, so a warp's
// store of one token is contiguous; warps 0-3 take the first half of the tile's tokens, 4-7
// the second; 16 warps were no faster), warp 8 loads, warp 9 issues. Three forms:
//  * kSingle: a CTA walks over tiles of 128 rows, the epilogue of one under the products of
//    the next (two accumulators);
//  * kPair: the same with the two SMs of a cluster on one tile of 256 rows (cta_group::2): each
//    loads its 128 weight rows and half of the tokens, a third less per SM and product than
//    kSingle's, which is bound by the loads from L2;
//  * kSplit: the CTAs of a cluster share one tile's K range, for products with few tiles; each
//    sends its sums to the CTA that owns the tokens, which adds them up (integers: the order
//    does not matter).
// Bound by the tensor pipe for large products (4096 x 7168 x 7168: 135 us = 3.1 POP/s for a burst; the
// pipe is busy for 90 % of the SMs' active cycles and 75 % of all, since 448 tiles on 74 pairs are six
// whole waves and one of 4 tiles), by the loads from L2 (about 100 bytes per ns
// and SM) and the stores for shallow ones (2047 x 1536 x 7168 into fp32: 26 us, 49 % active), and
// by the chain launch - quantise - load - join for small ones (64 x 5120 x 2304: 8.2 us).
enum : int { kSingle = 0, kPair = 1, kSplit = 2 };
constexpr int kGmEpiWarps = 8, kGmLoadWarp = kGmEpiWarps, kGmMmaWarp = kGmEpiWarps + 1;
constexpr int kGmThreads = 32 * (kGmEpiWarps + 2);
constexpr int kGmMaxStages = 12, kGmMaxSplit = 8;
constexpr int kGmABytes = 128 * 128;
constexpr int kGmSmem = 220 * 1024;           // dynamic shared memory, alignment included
constexpr uint32_t kGmTmemCols = 512, kGmAccCols = 256;
constexpr uint64_t kGmTimeoutNs = 1000000000; // a pipeline wait longer than this is an error
constexpr uint32_t kGmDrainPolls = 1u << 22;

struct Int8Gemm {
    CUtensorMap wmap, xmap;  // [n][k] box 128 rows, [tokens][k] box: a CTA's token rows; 128 bytes wide
    const float *w_scale, *q_scale, *bias;
    void* out;
    int* status;
    int64_t ld_out;
    int tokens, n, kblocks, nt, stages, ntiles, tiles, split;
    bool pairs;  // 16-bit outputs: two rows of a token in one aligned 4-byte store
};

// kSplit: the tokens of a tile that one CTA of the cluster adds up: whole fours, the last CTAs may
// have none.
__host__ __device__ constexpr int gm_share(int nt, int split) { return ((nt + split - 1) / split + 3) & ~3; }

// D (+)= A . B^T, both operands described in shared memory (PAIR: of both CTAs).
template <bool PAIR>
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// One arrival on `bar` (PAIR: on the barrier at that place in both CTAs) once the products
// issued so far have completed.
template <bool PAIR>
__device__ __forceinline__ void gm_commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        umma_commit(bar);
}
// A 2-D tile into this CTA; PAIR: counted on a barrier of the leading CTA.
template <bool PAIR>
__device__ __forceinline__ void gm_load(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
            "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        tma_2d(dst, map, x, y, bar);
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Waits for the loads; the registers pass through, so that no use of them moves in front.
__device__ __forceinline__ void tmem_wait16(int (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
// K-major operand, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61) |
           (uint64_t)((addr >> 4) & 0x3FFFu);
}
// Parity wait whose acquire covers the peer CTA's arrivals.
__device__ __forceinline__ bool mbar_try_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P1, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, P1;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(kTcSuspendNs)
        : "memory");
    return done != 0;
}
__device__ __noinline__ bool gm_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
    const uint64_t t0 = tc_now_ns();
    for (;;) {
        if (mbar_try_cluster(bar, parity)) return true;
        if (*abort_flag) return false;
        if (tc_now_ns() - t0 > kGmTimeoutNs) break;
    }
    if (status) atomicExch(status, kErrInt8Wait);
    *abort_flag = 1;
    return false;
}
__device__ __forceinline__ bool gm_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
    return mbar_try_cluster(bar, parity) || gm_wait_slow(bar, parity, abort_flag, status);
}

template <int OUT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if (OUT == CLB_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Sixteen tokens from t0 on of one warp's 32 rows (row: this lane's), from accumulators to
// the output. xs: the tokens' scales in shared memory.
template <int OUT>
__device__ __forceinline__ void gm_store16(const Int8Gemm& g, const int (&r)[16], const float* xs, int t0, int row, float ws,
                                           float bias) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(xs + j);
        v[j] = int8_value(r[j], x.x, ws, bias, true);
        v[j + 1] = int8_value(r[j + 1], x.y, ws, bias, true);
        v[j + 2] = int8_value(r[j + 2], x.z, ws, bias, true);
        v[j + 3] = int8_value(r[j + 3], x.w, ws, bias, true);
    }
    const int n = min(16, g.tokens - t0);
    if (OUT != CLB_F32 && g.pairs) {
        // even lanes take the even tokens of rows (row, row + 1), odd lanes the odd tokens of (row - 1, row)
        const bool odd = row & 1;
        uint16_t* p = static_cast<uint16_t*>(g.out) + (int64_t)(t0 + odd) * g.ld_out + (row & ~1);
        const bool ok = row < g.n;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
            const uint32_t w = odd ? pack16<OUT>(other, v[j + 1]) : pack16<OUT>(v[j], other);
            if (ok && j + odd < n) *reinterpret_cast<uint32_t*>(p) = w;
            p += 2 * g.ld_out;
        }
    } else if (row < g.n) {
        if (OUT == CLB_F32) {
            float* p = static_cast<float*>(g.out) + (int64_t)t0 * g.ld_out + row;
#pragma unroll
            for (int j = 0; j < 16; ++j, p += g.ld_out)
                if (j < n) *p = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < n) ops_store(g.out, OUT, (int64_t)(t0 + j) * g.ld_out + row, v[j]);
        }
    }
}

template <int MODE, int OUT>
__global__ void __launch_bounds__(kGmThreads, 1) k_int8_gemm(const __grid_constant__ Int8Gemm g) {
    constexpr bool PAIR = MODE == kPair, SPLIT = MODE == kSplit;
    extern __shared__ uint8_t gm_smem[];
    __shared__ __align__(16) float xs_s[2][kGmAccCols];
    __shared__ uint64_t bars[2 * kGmMaxStages + 5];
    __shared__ uint32_t tslot;
    __shared__ int abort_s;
    const uint32_t base = ((uint32_t)__cvta_generic_to_shared(gm_smem) + 1023u) & ~1023u;
    const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
    auto full = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    auto empty = [&](int i) { return bar0 + 8u * (uint32_t)(kGmMaxStages + i); };
    auto acc_full = [&](int i) { return bar0 + 8u * (uint32_t)(2 * kGmMaxStages + i); };
    auto acc_empty = [&](int i) { return bar0 + 8u * (uint32_t)(2 * kGmMaxStages + 2 + i); };
    const uint32_t drain = bar0 + 8u * (uint32_t)(2 * kGmMaxStages + 4);
    volatile int* abort_flag = &abort_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // this CTA's place in its cluster, the tiles it walks over, and its K blocks
    const int peers = PAIR ? 2 : SPLIT ? g.split : 1;
    const int rank = MODE == kSingle ? 0 : (int)blockIdx.x % peers;
    const int first = (int)blockIdx.x / peers, step = (int)gridDim.x / peers;
    const int my_tiles = SPLIT ? 1 : (g.tiles - 1 - first) / step + 1;
    const int kb0 = SPLIT ? (int)((int64_t)g.kblocks * rank / g.split) : 0;
    const int nkb = (SPLIT ? (int)((int64_t)g.kblocks * (rank + 1) / g.split) : g.kblocks) - kb0;
    const int64_t total = (int64_t)my_tiles * nkb;
    const int tile_rows = PAIR ? 256 : 128, brows = PAIR ? g.nt / 2 : g.nt;
    const uint32_t stage_bytes = (uint32_t)kGmABytes + (uint32_t)brows * 128u;
    // neighbours share the weights' rows (the other order: 143 us for 135 at 4096 x 7168 x 7168)
    auto row_of = [&](int tile) { return (tile / g.ntiles) * tile_rows + (PAIR ? 128 * rank : 0); };
    auto token_of = [&](int tile) { return (tile % g.ntiles) * g.nt; };

    if (tid == 32 * kGmLoadWarp) {
        for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(empty(i), 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full(i), 1), mbar_init(acc_empty(i), (PAIR ? 2 : 1) * kGmEpiWarps);
        mbar_init(drain, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        const uint32_t slot = (uint32_t)__cvta_generic_to_shared(&tslot);
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(kGmTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(kGmTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    // the peer's barriers and tensor memory are there
    if (PAIR) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    // weights do not depend on the quantising kernel in front, and what is in front of that is
    // complete (ops_begin): their first loads go out before that kernel has finished, the tokens' after
    const int ahead = (int)min((int64_t)g.stages, total);
    const uint32_t lead = PAIR ? cluster_addr(full(0), 0) : full(0);  // the stages' full barriers
    if (tid == 32 * kGmLoadWarp) {
        int tile = first, kb = 0, row = row_of(tile);
        for (int i = 0; i < ahead; ++i) {
            if (rank == 0 || !PAIR) mbar_expect_tx(full(i), (PAIR ? 2u : 1u) * stage_bytes);
            gm_load<PAIR>(base + (uint32_t)i * stage_bytes, &g.wmap, (kb0 + kb) * 128, row, lead + 8u * (uint32_t)i);
            if (++kb == nkb) kb = 0, tile += step, row = row_of(tile);
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (SPLIT) cluster_arrive();  // waited for before the first access to a peer
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tslot);
    // SPLIT: [source][four tokens of this CTA's share][128 rows][token] behind the stages, so that a
    // warp's rows send 512 bytes in a row (64 x 5120 x 2304: 8.3 us, 8.4 token by token, 9.4 with a
    // row's tokens together)
    const int share = SPLIT ? gm_share(g.nt, g.split) : 0;
    const uint32_t red = base + (uint32_t)g.stages * stage_bytes;
    float split_ws = 0.0f, split_bias = -0.0f;  // for the sums that this CTA will add up

    if (warp == kGmLoadWarp) {
        if (lane == 0) {
            ops_wait();
            // the place of a tile is found once a tile: the divisions in front of every copy would cost
            // more than the block's products
            int stage = 0, left = ahead;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = 0; i < my_tiles && ok; ++i) {
                const int row = row_of(first + i * step), token = token_of(first + i * step) + (PAIR ? brows * rank : 0);
                for (int x = kb0 * 128; x < (kb0 + nkb) * 128; x += 128) {
                    const uint32_t a = base + (uint32_t)stage * stage_bytes, bar = lead + 8u * (uint32_t)stage;
                    if (left > 0) {  // the weights are on their way
                        --left;
                    } else {
                        if (!(ok = gm_wait(empty(stage), phase ^ 1u, abort_flag, g.status))) break;
                        if (rank == 0 || !PAIR) mbar_expect_tx(full(stage), (PAIR ? 2u : 1u) * stage_bytes);
                        gm_load<PAIR>(a, &g.wmap, x, row, bar);
                    }
                    gm_load<PAIR>(a + kGmABytes, &g.xmap, x, token, bar);
                    if (++stage == g.stages) stage = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == kGmMmaWarp) {
        if (lane == 0 && (rank == 0 || !PAIR)) {
            // D s32, A and B signed 8-bit, N and M of the instruction
            const uint32_t idesc =
                (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(g.nt >> 3) << 17) | ((uint32_t)(tile_rows >> 4) << 24);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = 0; i < my_tiles && ok; ++i) {
                const int acc = i & 1;
                if (i >= 2 && !gm_wait(acc_empty(acc), (uint32_t)((i >> 1) & 1) ^ 1u, abort_flag, g.status)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!(ok = gm_wait(full(stage), phase, abort_flag, g.status))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a = base + (uint32_t)stage * stage_bytes;
                    const uint64_t da = smem_desc(a), db = smem_desc(a + kGmABytes);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        umma_i8<PAIR>(tmem + (uint32_t)acc * kGmAccCols, da + 2u * j, db + 2u * j, idesc, kb > 0 || j > 0);
                    gm_commit<PAIR>(empty(stage));
                    if (++stage == g.stages) stage = 0, phase ^= 1u;
                }
                if (ok) gm_commit<PAIR>(acc_full(acc));
            }
        }
    } else {
        ops_begin();  // q_scale
        const uint32_t tlane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        constexpr int kParts = kGmEpiWarps / 4;  // of the tile's tokens
        const int part = (g.nt / 16 + kParts - 1) / kParts * 16, c0 = min(g.nt, part * (warp >> 2)), c1 = min(g.nt, c0 + part);
        const uint32_t lead_empty = PAIR ? cluster_addr(acc_empty(0), 0) : 0u;
        bool ok = true;
        if (SPLIT) {
            const int row = row_of(first) + (tid & 127), t = token_of(first) + rank * share + tid;
            if (row < g.n) {
                split_ws = g.w_scale[row];
                if (g.bias) split_bias = g.bias[row];
            }
            if (tid < share) xs_s[0][tid] = t < g.tokens ? g.q_scale[t] : 0.0f;
            cluster_wait();
        }
        for (int i = 0; i < my_tiles; ++i) {  // to the end after a failed wait too: the warps meet at a barrier
            const int acc = i & 1, tile = first + i * step;
            const int row = row_of(tile) + (tid & 127), t0 = token_of(tile);
            float ws = 0.0f, bias = -0.0f;  // adding -0 leaves every number as it is
            if (!SPLIT) {
                if (tid < g.nt) xs_s[acc][tid] = t0 + tid < g.tokens ? g.q_scale[t0 + tid] : 0.0f;
                if (row < g.n) {
                    ws = g.w_scale[row];
                    if (g.bias) bias = g.bias[row];
                }
                // the scales of a tile are written once all warps have left the tile two before it
                asm volatile("bar.sync 1, %0;" ::"r"(32 * kGmEpiWarps) : "memory");
            }
            if (ok) ok = __all_sync(0xffffffffu, gm_wait(acc_full(acc), (uint32_t)(i >> 1) & 1u, abort_flag, g.status));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (ok) {
                const uint32_t ta = tlane + (uint32_t)acc * kGmAccCols;
                // SPLIT: where the sums of token c go
                int owner = SPLIT ? c0 / share : 0, off = SPLIT ? c0 % share : 0;
                auto send_to = [&] { return cluster_addr(red + (uint32_t)((rank * share + off) * 128 + 4 * (tid & 127)) * 4u, owner); };
                uint32_t to = SPLIT && c0 < c1 ? send_to() : 0u;
                auto take = [&](const int (&r)[16], int c) {
                    if (SPLIT) {
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(r[j]), "r"(r[j + 1]),
                                         "r"(r[j + 2]), "r"(r[j + 3])
                                         : "memory");
                            to += 2048u, off += 4;
                            if (off == share && c + j + 4 < g.nt) off = 0, ++owner, to = send_to();
                        }
                    } else if (t0 + c < g.tokens) {
                        gm_store16<OUT>(g, r, &xs_s[acc][c], t0 + c, row, ws, bias);
                    }
                };
                int ra[16], rb[16] = {};
                if (c0 < c1) tmem_ld16(ta + (uint32_t)c0, ra);
                for (int c = c0; c < c1; c += 32) {
                    tmem_wait16(ra);
                    if (c + 16 < c1) tmem_ld16(ta + (uint32_t)c + 16u, rb);
                    take(ra, c);
                    tmem_wait16(rb);
                    if (c + 32 < c1) tmem_ld16(ta + (uint32_t)c + 32u, ra);
                    if (c + 16 < c1) take(rb, c + 16);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (PAIR)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_empty + 8u * acc)
                                 : "memory");
                else
                    mbar_arrive(acc_empty(acc));
            }
        }
    }
    __syncwarp();

    if (SPLIT) {
        if (warp >= kGmEpiWarps) cluster_wait();
        cluster_arrive();
        cluster_wait();
        // every peer's sums are here: this CTA's share of the tile's tokens
        const int t0 = token_of(first) + rank * share, row = row_of(first) + (tid & 127);
        const int nc = min(share, min(g.nt - rank * share, g.tokens - t0));
        if (warp < kGmEpiWarps && row < g.n && !*abort_flag) {
            for (int c = 4 * (tid >> 7); c < nc; c += kGmEpiWarps) {
                int sum[4] = {};
#pragma unroll
                for (int p = 0; p < kGmMaxSplit; ++p) {
                    int v[4] = {};
                    if (p < g.split)
                        asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                                     : "r"(red + (uint32_t)((p * share + c) * 128 + 4 * (tid & 127)) * 4u));
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[j] += v[j];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < nc)
                        ops_store(g.out, OUT, (int64_t)(t0 + c + j) * g.ld_out + row,
                                  int8_value(sum[j], xs_s[0][c + j], split_ws, split_bias, true));
            }
        }
    }
    __syncthreads();
    if (*abort_flag) {  // let copies in flight land and the issued products complete before leaving
        const uint64_t t0 = tc_now_ns();
        while (tc_now_ns() - t0 < 200000u) {
        }
        if (warp == kGmMmaWarp && lane == 0 && (rank == 0 || !PAIR)) {
            gm_commit<PAIR>(drain);
            for (uint32_t i = 0; i < kGmDrainPolls && !mbar_try(drain, 0); ++i) {
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) {  // the peer's products and copies use this CTA's memory until both are done
        cluster_arrive();
        cluster_wait();
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kGmTmemCols));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kGmTmemCols));
    }
}

// The form of a product, by an estimate of its time (us): a 128-byte block of K costs its loads and, from
// about 100 token columns on, its multiply-adds; a tile a fixed part, a launch or a split another. CTAs
// run in waves over the SMs, clusters in the number that fits at once. The constants were fitted for 16
// to 128 tokens, and for larger products before neighbouring tiles shared the weights' rows: those it
// overstates (4096 x 7168 x 7168: 183 us for 135; 1024 x 7168 x 7168: 53 for 40; 2047 x 1536 x 7168: 28 for
// 25). Measured on a B200 (product alone, tokens a tile in brackets):
// 4096 x 7168 x 7168 single (256) 148 us, pair (256, chosen) 135, pair (224) 144; 1024 x 7168 x 7168 single
// (256) 47, pair (224, chosen) 40.0, pair (256) 41.3; 500 x 1536 x 7168 single (256) 9.5, pair (256, chosen) 10.5,
// single (128) 12.0; 64 x 5120 x 2304 (64) single 14.5, split in two 11.1, in four 8.8, in six (chosen) 8.2,
// in seven (more clusters than fit at once) 14.0; 64 x 512 x 2304 single (32, chosen) 4.9, single (64) 5.3,
// split in four 6.3.
struct GmPlan {
    int mode, nt, split;
};
struct GmDevice {
    int sms;
    int clusters[kGmMaxSplit + 1];  // clusters of that many CTAs that run at once
};

GmPlan gm_plan(int tokens, int n, int kblocks, const GmDevice& d) {
    GmPlan best{kSingle, 16, 1};
    double least = 1e300;
    auto consider = [&](int mode, int nt, int split) {
        const int64_t tiles = (int64_t)((n + (mode == kPair ? 255 : 127)) / (mode == kPair ? 256 : 128)) * ((tokens + nt - 1) / nt);
        const int64_t at_once = mode == kSingle ? d.sms : d.clusters[mode == kPair ? 2 : split];
        if (at_once < 1) return;
        const int64_t waves = (tiles + at_once - 1) / at_once;
        if (mode == kSplit && waves > 1) return;
        const double block = mode == kPair ? std::max(0.30, 0.241 + 0.00077 * nt) : std::max(0.29, 0.15 + 0.00139 * nt);
        const double blocks = (kblocks + split - 1) / split * block;
        const double full = std::min(1.0, (double)tiles / at_once);
        const double cost = mode == kSplit ? blocks + 5.4 + 0.02 * nt + 0.3 * full
                                           : waves * (blocks + 0.8) + 3.2 + 0.006 * nt + 0.6 * full;
        if (cost < least) least = cost, best = GmPlan{mode, nt, split};
    };
    for (int nt = 16; nt <= 256; nt += 16) {
        consider(kSingle, nt, 1);
        if (nt % 32 == 0) consider(kPair, nt, 1);
        for (int split = 2; split <= kGmMaxSplit && split <= kblocks && nt <= 128; ++split) consider(kSplit, nt, split);
        if (nt >= tokens) break;
    }
    return best;
}

cudaError_t gm_encode(CUtensorMap* map, const void* p, int64_t rows, int k, int64_t ld, int box_rows) {
    EncodeTiledFn encode = nullptr;
    const cudaError_t e = tc_encoder(&encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, es[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

template <int MODE>
void (*gm_kernel(int out_type))(Int8Gemm) {
    return out_type == CLB_F32 ? k_int8_gemm<MODE, CLB_F32> : out_type == CLB_BF16 ? k_int8_gemm<MODE, CLB_BF16>
                                                                                    : k_int8_gemm<MODE, CLB_F16>;
}
void (*gm_kernel(int mode, int out_type))(Int8Gemm) {
    return mode == kSingle ? gm_kernel<kSingle>(out_type) : mode == kPair ? gm_kernel<kPair>(out_type)
                                                                          : gm_kernel<kSplit>(out_type);
}

cudaError_t gm_launch(const Int8Gemm* g, int mode, int out_type, int clusters, int cluster, bool overlap, cudaStream_t s,
                      int* at_once) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)clusters * (unsigned)cluster);
    c.blockDim = dim3(kGmThreads);
    c.dynamicSmemBytes = kGmSmem;
    c.stream = s;
    c.attrs = attr;
    if (cluster > 1) {
        attr[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[c.numAttrs].val.clusterDim.x = (unsigned)cluster;
        attr[c.numAttrs].val.clusterDim.y = attr[c.numAttrs].val.clusterDim.z = 1;
        ++c.numAttrs;
    }
    if (at_once) return cudaOccupancyMaxActiveClusters(at_once, gm_kernel(mode, out_type), &c);
    if (overlap) {
        attr[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++c.numAttrs;
    }
    return cudaLaunchKernelEx(&c, gm_kernel(mode, out_type), *g);
}

// The current device: its SMs and the clusters they hold (found once, with the kernels' shared
// memory allowed).
cudaError_t gm_device(const GmDevice** out) {
    static GmDevice devices[64];
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    e = ops_device(&sms, [&] {
        GmDevice& d = devices[dev];
        cudaError_t e;
        if ((e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
        for (int mode = kSingle; mode <= kSplit; ++mode)
            for (int type : {CLB_F32, CLB_BF16, CLB_F16})
                if ((e = cudaFuncSetAttribute(gm_kernel(mode, type), cudaFuncAttributeMaxDynamicSharedMemorySize, kGmSmem)) !=
                    cudaSuccess)
                    return e;
        for (int tt : {1, 2, 4})
            for (bool vec : {false, true})
                for (int type : {CLB_F32, CLB_BF16, CLB_F16})
                    if ((e = cudaFuncSetAttribute(dot_kernel(tt, vec, type), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  kDotSmemMax)) != cudaSuccess)
                        return e;
        for (int size = 2; size <= kGmMaxSplit; ++size)
            if ((e = gm_launch(nullptr, size == 2 ? kPair : kSplit, CLB_F32, 1, size, false, nullptr, &d.clusters[size])) !=
                cudaSuccess)
                return e;
        return cudaSuccess;
    });
    *out = &devices[dev];
    return e;
}

cudaError_t launch_int8_gemm(const Int8Args& a, int* status, bool overlap, const GmDevice& d, cudaStream_t s) {
    cudaError_t e;
    Int8Gemm g{};
    g.kblocks = (a.k + 127) / 128;
    const GmPlan plan = gm_plan(a.tokens, a.n, g.kblocks, d);
    const bool pair = plan.mode == kPair;
    const int brows = pair ? plan.nt / 2 : plan.nt;
    g.nt = plan.nt, g.split = plan.split;
    if ((e = gm_encode(&g.wmap, a.w, a.n, a.k, a.ld_w, 128)) != cudaSuccess) return e;
    if ((e = gm_encode(&g.xmap, a.q, a.tokens, a.k, a.ld_q, brows)) != cudaSuccess) return e;
    g.w_scale = a.w_scale, g.q_scale = a.q_scale, g.bias = a.bias, g.out = a.out, g.status = status;
    g.ld_out = a.ld_out, g.tokens = a.tokens, g.n = a.n;
    g.pairs = a.n % 2 == 0 && a.ld_out % 2 == 0 && ops_aligned(a.out, 4);
    const int joined = plan.mode == kSplit ? plan.split * 512 * gm_share(plan.nt, plan.split) : 0;  // the peers' sums
    g.stages = std::min(kGmMaxStages, (kGmSmem - 1024 - joined) / (kGmABytes + brows * 128));
    g.ntiles = (a.tokens + g.nt - 1) / g.nt;
    g.tiles = (a.n + (pair ? 255 : 127)) / (pair ? 256 : 128) * g.ntiles;
    const int at_once = pair ? d.clusters[2] : d.sms;
    return gm_launch(&g, plan.mode, a.out_type, plan.mode == kSplit ? g.tiles : std::min(g.tiles, at_once),
                     pair ? 2 : plan.split, overlap, s, nullptr);
}

// Up to this many tokens the product is row dots, above it (or when the quantised tokens do
// not fit in shared memory) tensor-core tiles.
constexpr int kDotTokens = 4;

cudaError_t launch_int8_dot(const Int8Args& a, const void* x, int x_type, int64_t ld_x, const GmDevice& dev, cudaStream_t s) {
    Int8Dot d{a, x, ld_x, 0, 0, (a.k + 15) & ~15};
    const bool vec = !x || ops_vec8(x, x_type, ld_x);
    const int tt = a.tokens <= 1 ? 1 : a.tokens <= 2 ? 2 : 4;
    d.rows = std::min((a.n + dev.sms - 1) / dev.sms, kDotMaxSums / tt);
    // cut the rows so that the warps' shares are even; an item costs its groups and as much as half a
    // group for its sums
    double least = 1e300;
    for (int log = 0; log <= 5 && (d.kpad >> log) >= 512; ++log) {
        const int per = ((a.k >> 4) + (1 << log) - 1) >> log, groups = (per + 32 * kDotAhead - 1) / (32 * kDotAhead);
        const double cost = (double)(((d.rows << log) + kDotThreads / 32 - 1) / (kDotThreads / 32)) * (groups + 0.5);
        if (cost < least) least = cost, d.log_segs = log;
    }
    void (*kernel)(Int8Dot) = dot_kernel(tt, vec, x ? x_type : CLB_F32);
    const size_t smem = (size_t)tt * d.kpad + (size_t)d.rows * tt * 4;
    return ops_launch(kernel, (unsigned)((a.n + d.rows - 1) / d.rows), kDotThreads, smem, s, d);
}
bool dot_fits(int tokens, int k) {
    const int tt = tokens <= 1 ? 1 : tokens <= 2 ? 2 : 4;
    return tokens <= kDotTokens && (int64_t)tt * ((k + 15) & ~15) <= kDotSmem;
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
        const clb::OpsRows in[] = {clb::ops_rows("x", d_x, rows, k, ld_x, type)};
        const clb::OpsRows q = clb::ops_rows("q", d_q, rows, k, ld_q, CLB_I8);
        const clb::OpsRows scale = clb::ops_rows("scale", d_scale, 1, rows, rows, CLB_F32), to_scale[] = {scale};
        clb::ops_require_apart(q, in);
        clb::ops_require_apart(scale, in);
        clb::ops_require_apart(q, to_scale);
        cuda_check(clb::launch_int8_quantize(d_x, type, ld_x, rows, k, d_q, ld_q, k, d_scale,
                                             static_cast<cudaStream_t>(stream)),
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
        require(c.n >= 1 && c.n <= clb::kInt8MaxRows && c.k >= 1 && c.k <= clb::kInt8MaxK, CLB_E_INVALID,
                "n in 1..%d and k in 1..%d", clb::kInt8MaxRows, clb::kInt8MaxK);
        require((ready || clb::ops_float_type(c.x_type)) && clb::ops_float_type(c.out_type), CLB_E_INVALID,
                "x is fp32, bf16, fp16 or int8; out is fp32, bf16 or fp16");
        require(c.ld_w >= c.k && c.ld_w % 16 == 0, CLB_E_INVALID, "ld_w is a multiple of 16, at least k");
        require(c.ld_x >= c.k && (!ready || c.ld_x % 16 == 0), CLB_E_INVALID,
                "ld_x is at least k (a multiple of 16 for int8)");
        require(c.ld_out >= c.n, CLB_E_INVALID, "ld_out below n");
        for (int i = 0; i < 4; ++i) require(!c.reserved[i], CLB_E_INVALID, "reserved fields must be 0");
        require(tokens >= 0 && tokens <= clb::kInt8MaxRows, CLB_E_INVALID, "token count not in 0..%d", clb::kInt8MaxRows);
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
        const int64_t ws_need = ready ? 0 : (int64_t)clb_int8_linear_workspace_bytes(tokens, c.k);
        const clb::OpsRows ws = clb::ops_rows("the workspace", ready ? nullptr : d_ws, 1, ws_need, ws_need, CLB_I8), to_ws[] = {ws};
        const clb::OpsRows in[] = {clb::ops_rows("x", d_x, tokens, c.k, c.ld_x, c.x_type),
                                   clb::ops_rows("x_scale", d_x_scale, 1, tokens, tokens, CLB_F32),
                                   clb::ops_rows("w", d_w, c.n, c.k, c.ld_w, CLB_I8),
                                   clb::ops_rows("w_scale", d_w_scale, 1, c.n, c.n, CLB_F32),
                                   clb::ops_rows("bias", d_bias, 1, c.n, c.n, CLB_F32)};
        const clb::OpsRows out = clb::ops_rows("out", d_out, tokens, c.n, c.ld_out, c.out_type);
        clb::ops_require_apart(out, in);
        clb::ops_require_apart(out, to_ws);
        clb::ops_require_apart(ws, in);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        clb::Int8Args a{d_w, nullptr, d_w_scale, nullptr, d_bias, d_out, c.ld_w, 0, c.ld_out, tokens, c.n, c.k,
                        c.out_type};
        if (ready) {
            a.q = static_cast<const int8_t*>(d_x);
            a.q_scale = d_x_scale;
            a.ld_q = c.ld_x;
        }
        const clb::GmDevice* device = nullptr;
        cuda_check(clb::gm_device(&device), "int8 product set-up");
        if (clb::dot_fits(tokens, c.k)) {
            cuda_check(clb::launch_int8_dot(a, ready ? nullptr : d_x, c.x_type, c.ld_x, *device, s), "int8 row dots");
            return;
        }
        if (!ready) {
            a.ld_q = clb::round16(c.k);
            float* scale = reinterpret_cast<float*>(static_cast<int8_t*>(d_ws) + tokens * a.ld_q);
            a.q = static_cast<const int8_t*>(d_ws);
            a.q_scale = scale;
            cuda_check(clb::launch_int8_quantize(d_x, c.x_type, c.ld_x, tokens, c.k, static_cast<int8_t*>(d_ws), a.ld_q,
                                                 (int)a.ld_q, scale, s),
                       "int8 quantise");
        }
        cuda_check(clb::launch_int8_gemm(a, d_status, !ready, *device, s), "int8 product");
    });
}
