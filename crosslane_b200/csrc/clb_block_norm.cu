// The residual step between two blocks: RMSNorm after the block, gate, scaled residual sum,
// RMSNorm before the next block, in one pass over the rows: y and h are read once, h' and x
// written once, so the kernels are bound by those bytes. A CTA holds a row in registers. The
// two sums of squares are fp32: per thread in element order (one chain, or one for the even
// and one for the odd elements), then over the warp and the CTA in a fixed tree.
#include <algorithm>
#include <cmath>

#include "clb_ops.cuh"
#include "clb_tc.cuh"

namespace clb {
namespace {

constexpr int kNormMaxDim = 32768;
constexpr int64_t kNormManyChunks = 200000;  // rows * chunks of 8 from which k_block_norm_rows is faster
constexpr int kRowFlight = 104 * 1024, kRowFlightTwo = 132 * 1024;  // bytes of rows asked for ahead on an SM
constexpr int kRowSmem = 216 * 1024;    // the most a single CTA's rows take

struct NormArgs {
    const void *h, *y, *gate;
    const float *w_post, *w_pre;
    void *h_out, *x;
    int64_t ld_h, ld_y, ld_gate, ld_h_out, ld_x;
    int tokens, dim, h_type, y_type, gate_type, x_type, gate_kind, gate_sigmoid, post;
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

// Eight values of a thread's chunk c. W 8: 8 contiguous elements, 16- and 32-byte accesses. W 4, 2: two
// fours or four pairs, blockDim of them apart (the elements behind the last whole one are single
// values of the first threads). W 1: elements, blockDim apart. So a warp's accesses are contiguous.
template <int W>
__device__ __forceinline__ Raw8 load8(const void* p, int type, int64_t row, int c, int dim) {
    const char* r = static_cast<const char*>(p) + row * (type == CLB_F32 ? 4 : 2);
    const int nt = blockDim.x, tid = threadIdx.x;
    if (W == 8) return raw8_aligned(r, type, 8 * (int64_t)(tid + c * nt), tid + c * nt < dim >> 3);
    if (W == 1) return raw8_strided(r, type, 8 * (int64_t)c * nt + tid, nt, dim);
    Raw8 v{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (W == 2) {
        uint32_t w[8] = {};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = (4 * c + k) * nt + tid;
            const bool ok = i < dim >> 1;
            uint32_t pair = 0;
            ld8_if(w[2 * k], w[2 * k + 1], r + 8 * (int64_t)i, ok && type == CLB_F32);
            ld4_if(pair, r + 4 * (int64_t)i, ok && type != CLB_F32);
            if (type != CLB_F32) (&v.a.x)[k] = pair;
        }
        return type == CLB_F32 ? Raw8{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])} : v;
    }
    const int i = 2 * c * nt + tid, j = i + nt, n = dim >> 2;
    ld16_if(v.a, r + 16 * (int64_t)i, i < n && type == CLB_F32);
    ld16_if(v.b, r + 16 * (int64_t)j, j < n && type == CLB_F32);
    ld8_if(v.a.x, v.a.y, r + 8 * (int64_t)i, i < n && type != CLB_F32);
    ld8_if(v.a.z, v.a.w, r + 8 * (int64_t)j, j < n && type != CLB_F32);
    return v;
}
template <int W>
__device__ __forceinline__ void store8(void* p, int type, int64_t row, int c, int dim, const float (&v)[8]) {
    const int nt = blockDim.x, tid = threadIdx.x;
    if (W == 8) {
        if (tid + c * nt < dim >> 3) store8_aligned(p, type, row + 8 * (int64_t)(tid + c * nt), v);
    } else if (W == 4) {
        const int i = 2 * c * nt + tid, j = i + nt, n = dim >> 2;
        if (type == CLB_F32) {
            float4* r = reinterpret_cast<float4*>(static_cast<float*>(p) + row);
            if (i < n) r[i] = make_float4(v[0], v[1], v[2], v[3]);
            if (j < n) r[j] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint2* r = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + row);
            const uint4 w = pack8(type, v);
            if (i < n) r[i] = make_uint2(w.x, w.y);
            if (j < n) r[j] = make_uint2(w.z, w.w);
        }
    } else if (W == 2) {
        const uint4 packed = pack8(type, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = (4 * c + k) * nt + tid;
            if (i >= dim >> 1) continue;
            if (type == CLB_F32) reinterpret_cast<float2*>(static_cast<float*>(p) + row)[i] = make_float2(v[2 * k], v[2 * k + 1]);
            else reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + row)[i] = (&packed.x)[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = (c * 8 + j) * nt + tid;
            if (e < dim) ops_store(p, type, row + e, v[j]);
        }
    }
}

// sigmoid: expf and a reciprocal within 2 ulp each (a gate below -87.3, whose sigmoid is under
// 2^-126, is 0).
__device__ __forceinline__ float gate_value(float g, int sigmoid) {
    return sigmoid ? __fdividef(1.0f, 1.0f + expf(-g)) : g;
}

// The element types of a call as constants where they are a usual set (told apart at run time,
// they cost a bandwidth-bound kernel in 16 bits a third of its rate).
enum : int { kTypesAny = 0, kTypesF32, kTypesBF16, kTypesF16, kTypesF32BF16, kTypesF32F16 };  // the last two: h fp32
struct NormTypes {
    int h, other;
};
__host__ __device__ constexpr NormTypes norm_types(int set) {
    return set == kTypesF32    ? NormTypes{CLB_F32, CLB_F32}
           : set == kTypesBF16 ? NormTypes{CLB_BF16, CLB_BF16}
           : set == kTypesF16  ? NormTypes{CLB_F16, CLB_F16}
           : set == kTypesF32BF16 ? NormTypes{CLB_F32, CLB_BF16}
                                  : NormTypes{CLB_F32, CLB_F16};
}

// One CTA per row, CH chunks of 8 values per thread: few rows, where the latency of one counts (up
// to 1.6 million values: 200 x 7168 fp32 6.4 us, with k_block_norm_rows 7.0; 400 x 7168 12.7 and
// 11.5 us; 1200 x 1024 fp32 / bf16 3.9 and 5.5 us; 2000 x 1024 5.7 and 5.9 us),
// rows that are not aligned, and rows too wide for k_block_norm_rows. Bound by the latency of the
// loads and the two sums. Measured on a B200 (device time): 1 x 7168 fp32 3.2 us, 64 x 7168
// 3.6 us, 777 x 2311 fp32 / fp16 in rows of 2316 elements 4.4 us (4.9 TB/s; 6.8 element by element,
// the way of rows of odd pitches), 2000 x 2311 bf16 12.5 and 20 us; in pairs 6313 x 822 fp16 16.8
// and 21.5 us. Rows wider than 16384 take four chunks a thread, whose registers spill (16 to 700 bytes a
// thread by layout and types), and one CTA an SM: 512 x 16384 bf16 17.5 us (k_block_norm_rows), 512 x
// 16392 31 us, 512 x 32768 43 us, fp32 72 us (3.7 TB/s).
template <int CH, int W, int SET, bool SHORT>
__global__ void __launch_bounds__(SHORT ? 256 : 1024) k_block_norm(const NormArgs a) {
    const int h_type = SET ? norm_types(SET).h : a.h_type, y_type = SET ? norm_types(SET).other : a.y_type;
    const int x_type = SET ? norm_types(SET).other : a.x_type;
    __shared__ float part[2][32];
    ops_begin();
    // SHORT: eight rows a CTA have a warp each and do not meet
    const int64_t row = SHORT ? (int64_t)blockIdx.x * 8 + threadIdx.y : blockIdx.x;
    if (SHORT && row >= a.tokens) return;
    auto row_sum = [&](float v, float* p) { return SHORT ? ops_warp_sum(v) : cta_sum(v, p); };
    const bool wide_gate = a.gate_kind == CLB_GATE_CHANNEL || a.gate_kind == CLB_GATE_FULL;
    Raw8 yr[CH], hr[CH], gr[CH];
    // W 4, 2: the element behind the whole fours or pairs that is this thread's, as it lies in memory
    constexpr bool PARTS = W == 4 || W == 2;
    const int last = (a.dim & -W) + threadIdx.x;
    const bool tail = PARTS && last < a.dim;
    uint32_t y1 = 0, h1 = 0, g1 = 0;
    float v[CH][8];
    if (a.y)
#pragma unroll
        for (int c = 0; c < CH; ++c) yr[c] = load8<W>(a.y, y_type, row * a.ld_y, c, a.dim);
#pragma unroll
    for (int c = 0; c < CH; ++c) hr[c] = load8<W>(a.h, h_type, row * a.ld_h, c, a.dim);
    if (PARTS) {
        ld_elem_if(y1, a.y, y_type, row * a.ld_y + last, tail && a.y);
        ld_elem_if(h1, a.h, h_type, row * a.ld_h + last, tail);
        ld_elem_if(g1, a.gate, a.gate_type, (a.gate_kind == CLB_GATE_FULL ? row * a.ld_gate : 0) + last, tail && wide_gate);
    }
    float v1 = elem_float(h1, h_type);
    if (CH == 1 && wide_gate) gr[0] = load8<W>(a.gate, a.gate_type, a.gate_kind == CLB_GATE_FULL ? row * a.ld_gate : 0, 0, a.dim);
    if (a.y) {
        float gt = 1.0f;
        if (a.gate_kind == CLB_GATE_TOKEN) gt = gate_value(ops_load(a.gate, a.gate_type, row), a.gate_sigmoid);
        float inv = 1.0f;
        if (a.post) {
            float ss = elem_float(y1, y_type) * elem_float(y1, y_type), y[8];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                raw8_floats(yr[c], y_type, W > 1, y);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
            }
            inv = rsqrtf(row_sum(ss, part[0]) * a.inv_dim + a.post_eps);
        }
        const float f = a.block_scale * gt * inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float y[8], w[8];
            raw8_floats(yr[c], y_type, W > 1, y);
            if (a.w_post) {
                raw8_floats(load8<W>(a.w_post, CLB_F32, 0, c, a.dim), CLB_F32, W > 1, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] *= w[j];
            }
            if (wide_gate) {
                if (CH > 1) gr[c] = load8<W>(a.gate, a.gate_type, a.gate_kind == CLB_GATE_FULL ? row * a.ld_gate : 0, c, a.dim);
                raw8_floats(gr[c], a.gate_type, W > 1, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] *= gate_value(w[j], a.gate_sigmoid);
            }
            raw8_floats(hr[c], h_type, W > 1, v[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = fmaf(f, y[j], a.residual_scale * v[c][j]);
            store8<W>(a.h_out, h_type, row * a.ld_h_out, c, a.dim, v[c]);
        }
        if (tail) {
            float y = elem_float(y1, y_type);
            if (a.w_post) y *= a.w_post[last];
            if (wide_gate) y *= gate_value(elem_float(g1, a.gate_type), a.gate_sigmoid);
            v1 = fmaf(f, y, a.residual_scale * v1);
            ops_store(a.h_out, h_type, row * a.ld_h_out + last, v1);
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) raw8_floats(hr[c], h_type, W > 1, v[c]);
    }
    if (a.x) {
        float ss = tail ? v1 * v1 : 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(v[c][j], v[c][j], ss);
        const float inv = rsqrtf(row_sum(ss, part[1]) * a.inv_dim + a.pre_eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float w[8];
            if (a.w_pre) raw8_floats(load8<W>(a.w_pre, CLB_F32, 0, c, a.dim), CLB_F32, W > 1, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = a.w_pre ? w[j] * (v[c][j] * inv) : v[c][j] * inv;
            store8<W>(a.x, x_type, row * a.ld_x, c, a.dim, w);
        }
        if (tail) ops_store(a.x, x_type, row * a.ld_x + last, a.w_pre ? a.w_pre[last] * (v1 * inv) : v1 * inv);
    }
}

// Many rows: CTAs that stay and walk over the rows. Bulk copies bring the next rows of y, h and
// a full gate into shared memory while one is worked on, so that HBM is busy all the time;
// what all rows share (w_post times the channels' gate, w_pre) stays in registers (from L1 it
// cost 72 us for 42). A row's shared memory is asked for again as soon as the CTA has read it.
// The instructions a thread spends on the two sums are as many as on 20 values, so it takes
// several chunks where the rows have them, several CTAs an SM hide the sums' latency, and the
// arithmetic is done in pairs. Measured on a B200 (device time): 2048 x 7168 fp32 38.9 us (6.0
// TB/s), 8192 x 5120 bf16 with a sigmoid gate 67 us (6.25 TB/s, 96 % of a copy's rate); a CTA per
// row took 65 and 138 us.
constexpr int kRowStages = 2;
constexpr uint32_t kRowPolls = 1u << 20;  // waits for a copy, each with a suspend hint of 20 us

// The gates of two values. FAST: exp2 of the scaled argument and a reciprocal, the instructions
// alone: off by at most (|g| + 8) half ulps of fp32, far below a half step of the 16-bit types
// that the call's results are rounded to (8192 x 5120 in a stream: 75 us with expf, 70 us so).
template <bool FAST>
__device__ __forceinline__ F2 gate2(F2 g, int sigmoid) {
    if (!sigmoid) return g;
    if (!FAST) {
        const float2 v = f2_floats(g);
        return f2(gate_value(v.x, 1), gate_value(v.y, 1));
    }
    const float2 t = f2_floats(f2_mul(g, f2(-1.44269504f, -1.44269504f)));
    float a, b;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(t.y));
    const float2 d = f2_floats(f2_add(f2(a, b), f2(1.0f, 1.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(d.y));
    return f2(a, b);
}

// Eight values, number i of a row in shared memory, as pairs.
__device__ __forceinline__ void row8(uint32_t p, int type, int i, F2 (&v)[4]) {
    Raw8 r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    const uint32_t at = p + (uint32_t)i * (type == CLB_F32 ? 32u : 16u);
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w) : "r"(at));
    if (type == CLB_F32)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                     : "r"(at + 16u));
    float w[8];
    raw8_floats(r, type, true, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2(w[2 * j], w[2 * j + 1]);
}
__device__ __forceinline__ void store8_pairs(void* p, int type, int64_t i, const F2 (&v)[4]) {
    float w[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = f2_floats(v[j]);
        w[2 * j] = f.x, w[2 * j + 1] = f.y;
    }
    store8_aligned(p, type, i, w);
}
// The sum of squares of eight values, in two chains (even and odd ones).
__device__ __forceinline__ void square_sum(F2& s, const F2 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s = f2_fma(v[j], v[j], s);
}
__device__ __forceinline__ float both(F2 s) {
    const float2 f = f2_floats(s);
    return f.x + f.y;
}

template <int CH, int THREADS, int CTAS, int SET>
__global__ void __launch_bounds__(THREADS, CTAS) k_block_norm_rows(const NormArgs a, int rows, int stages, uint32_t y_bytes,
                                                                   uint32_t h_bytes, uint32_t g_bytes) {
    constexpr bool FAST = SET == kTypesBF16 || SET == kTypesF16;  // the results have 16 bits
    extern __shared__ __align__(16) uint8_t row_smem[];
    __shared__ float part[4][32];
    __shared__ uint64_t bars[kRowStages];
    ops_begin();
    const int h_type = SET ? norm_types(SET).h : a.h_type, y_type = SET ? norm_types(SET).other : a.y_type;
    const int x_type = SET ? norm_types(SET).other : a.x_type, g_type = SET ? norm_types(SET).other : a.gate_type;
    const int tid = threadIdx.x, nt = blockDim.x, units = a.dim >> 3;
    const uint32_t stage_bytes = y_bytes + h_bytes + g_bytes;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(row_smem), bar0 = (uint32_t)__cvta_generic_to_shared(bars);
    auto at = [](const void* p, int type, int64_t i) { return static_cast<const char*>(p) + i * (type == CLB_F32 ? 4 : 2); };
    auto fetch = [&](int64_t row, int stage) {
        const uint32_t dst = base + (uint32_t)stage * stage_bytes, bar = bar0 + 8u * (uint32_t)stage;
        mbar_expect_tx(bar, stage_bytes);
        if (y_bytes) bulk_g2s(dst, at(a.y, y_type, row * a.ld_y), y_bytes, bar);
        bulk_g2s(dst + y_bytes, at(a.h, h_type, row * a.ld_h), h_bytes, bar);
        if (g_bytes) bulk_g2s(dst + y_bytes + h_bytes, at(a.gate, g_type, row * a.ld_gate), g_bytes, bar);
    };
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(bar0 + 8u * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int s = 0; s < stages; ++s)
            if (blockIdx.x + (int64_t)s * gridDim.x < rows) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    }
    F2 wp[CH][4], wq[CH][4];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float p[8], q[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = q[j] = 1.0f;
        if (a.w_post) raw8_floats(load8<8>(a.w_post, CLB_F32, 0, c, a.dim), CLB_F32, true, p);
        if (a.w_pre) raw8_floats(load8<8>(a.w_pre, CLB_F32, 0, c, a.dim), CLB_F32, true, q);
        if (a.gate_kind == CLB_GATE_CHANNEL) {
            raw8_floats(load8<8>(a.gate, a.gate_type, 0, c, a.dim), a.gate_type, true, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] *= gate_value(g[j], a.gate_sigmoid);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) wp[c][j] = f2(p[2 * j], p[2 * j + 1]), wq[c][j] = f2(q[2 * j], q[2 * j + 1]);
    }
    const F2 keep = f2(a.residual_scale, a.residual_scale);
    __syncthreads();
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (uint32_t row = blockIdx.x; row < (uint32_t)rows; row += gridDim.x) {
        float gt = a.block_scale;
        if (a.gate_kind == CLB_GATE_TOKEN) gt *= gate_value(ops_load(a.gate, a.gate_type, row), a.gate_sigmoid);
        bool here = mbar_try(bar0 + 8u * stage, phase);
        for (uint32_t i = 0; !here && i < kRowPolls; ++i) here = mbar_try_sleep(bar0 + 8u * stage, phase);
        const uint32_t sy = base + (uint32_t)stage * stage_bytes, sh = sy + y_bytes, sg = sh + h_bytes;
        // a copy that never came (the wait ran out) shows as a row of NaN
        const float ok = here ? 1.0f : __int_as_float(0x7fffffff);
        F2 v[CH][4];
        if (y_bytes) {
            float f = gt * ok;
            if (a.post) {
                F2 ss = 0, y[4];  // two zeros
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (tid + c * nt < units) {
                        row8(sy, y_type, tid + c * nt, y);
                        square_sum(ss, y);
                    }
                f *= rsqrtf(cta_sum(both(ss), part[2 * turn]) * a.inv_dim + a.post_eps);
            }
            const F2 ff = f2(f, f);
            char* out = const_cast<char*>(at(a.h_out, h_type, row * a.ld_h_out));
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int u = tid + c * nt;
                if (u < units) {
                    F2 y[4], g[4];
                    row8(sy, y_type, u, y);
                    row8(sh, h_type, u, v[c]);
                    if (g_bytes) {
                        row8(sg, g_type, u, g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = f2_mul(y[j], gate2<FAST>(g[j], a.gate_sigmoid));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[c][j] = f2_fma(ff, f2_mul(y[j], wp[c][j]), f2_mul(keep, v[c][j]));
                    store8_pairs(out, h_type, 8 * u, v[c]);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (tid + c * nt < units) row8(sh, h_type, tid + c * nt, v[c]);
        }
        float inv = ok;
        if (a.x) {
            F2 ss = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (tid + c * nt < units) square_sum(ss, v[c]);
            inv *= rsqrtf(cta_sum(both(ss), part[2 * turn + 1]) * a.inv_dim + a.pre_eps);
        } else {
            __syncthreads();
        }
        // the CTA has read the stage
        if (tid == 0 && row + (int64_t)stages * gridDim.x < rows) fetch(row + (int64_t)stages * gridDim.x, stage);
        if (a.x) {
            const F2 ii = f2(inv, inv);
            char* out = const_cast<char*>(at(a.x, x_type, row * a.ld_x));
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int u = tid + c * nt;
                if (u < units) {
                    F2 w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = f2_mul(wq[c][j], f2_mul(v[c][j], ii));
                    store8_pairs(out, x_type, 8 * u, w);
                }
            }
        }
        turn ^= 1;  // a row may have one sum and so one barrier only: rows take turns with the buffers
        if (++stage == stages) stage = 0, phase ^= 1u;
    }
}

template <int SET>
void (*rows_kernel(int ch, int threads))(NormArgs, int, int, uint32_t, uint32_t, uint32_t) {
    return ch == 1   ? (threads <= 32 ? k_block_norm_rows<1, 32, 16, SET> : k_block_norm_rows<1, 1024, 1, SET>)
           : ch == 2 ? (threads <= 32    ? k_block_norm_rows<2, 32, 16, SET>
                        : threads <= 352 ? k_block_norm_rows<2, 352, 2, SET>
                                         : k_block_norm_rows<2, 448, 2, SET>)
                     : (threads <= 256 ? k_block_norm_rows<4, 256, 2, SET> : k_block_norm_rows<4, 512, 1, SET>);
}

decltype(rows_kernel<kTypesAny>(0, 0)) rows_kernel(int set, int ch, int threads) {
    return set == kTypesF32       ? rows_kernel<kTypesF32>(ch, threads)
           : set == kTypesBF16    ? rows_kernel<kTypesBF16>(ch, threads)
           : set == kTypesF16     ? rows_kernel<kTypesF16>(ch, threads)
           : set == kTypesF32BF16 ? rows_kernel<kTypesF32BF16>(ch, threads)
           : set == kTypesF32F16  ? rows_kernel<kTypesF32F16>(ch, threads)
                                  : rows_kernel<kTypesAny>(ch, threads);
}

template <int W, int SET>
void (*row_kernel(int ch))(NormArgs) {  // ch 0: short rows
    return ch == 0   ? k_block_norm<1, W, SET, true>
           : ch == 1 ? k_block_norm<1, W, SET, false>
           : ch == 2 ? k_block_norm<2, W, SET, false>
                     : k_block_norm<4, W, SET, false>;
}
template <int SET>
void (*row_kernel(int ch, int width))(NormArgs) {
    return width == 8   ? row_kernel<8, SET>(ch)
           : width == 4 ? row_kernel<4, SET>(ch)
           : width == 2 ? row_kernel<2, SET>(ch)
                        : row_kernel<1, SET>(ch);
}
void (*row_kernel(int set, int ch, int width))(NormArgs) {
    return set == kTypesF32       ? row_kernel<kTypesF32>(ch, width)
           : set == kTypesBF16    ? row_kernel<kTypesBF16>(ch, width)
           : set == kTypesF16     ? row_kernel<kTypesF16>(ch, width)
           : set == kTypesF32BF16 ? row_kernel<kTypesF32BF16>(ch, width)
           : set == kTypesF32F16  ? row_kernel<kTypesF32F16>(ch, width)
                                  : row_kernel<kTypesAny>(ch, width);
}

// width: elements that every row's accesses may take at a time (8 also divides dim then).
cudaError_t launch_block_norm(const NormArgs& a, int tokens, int width, cudaStream_t s) {
    const int units = (a.dim + 7) / 8;
    const uint32_t y_bytes = a.y ? a.dim * ops_type_bytes(a.y_type) : 0, h_bytes = a.dim * ops_type_bytes(a.h_type);
    const uint32_t g_bytes = a.gate_kind == CLB_GATE_FULL ? a.dim * ops_type_bytes(a.gate_type) : 0;
    const uint32_t stage = y_bytes + h_bytes + g_bytes;
    int set = kTypesAny;
    for (int i = kTypesF32; i <= kTypesF32F16; ++i) {
        const NormTypes t = norm_types(i);
        if (a.h_type == t.h && (!a.y || a.y_type == t.other) && (!a.x || a.x_type == t.other) &&
            (!g_bytes || a.gate_type == t.other))
            set = i;
    }
    if (width == 8 && (int64_t)tokens * units > kNormManyChunks && units <= 2048 && 2 * stage <= (uint32_t)kRowSmem) {
        // Two rows in flight for each CTA, and as many CTAs as bring that to 104 KB an SM, or two up to 132 KB:
        // with more, reads and writes get into each other's way in HBM (8192 x 5120 bf16, gate: 66.6 us
        // with 123 KB, 76 us with 184 KB; 8192 x 2048 fp32 / bf16: 35.0 us with 98 KB, 38.9 us with 123
        // KB). Chunks a thread: 4 where rows are short; 2 for two CTAs with wide rows (the gated case with
        // 4: 84 us); 1 for a single CTA, which has to hide its sums by itself (2048 x 7168 fp32: 39.5 us,
        // with 2 41.0, with 4 42.0 us).
        int ctas = std::min(16, kRowFlight / 2 / (int)stage);
        if (ctas < 2) ctas = 4 * (int)stage <= kRowFlightTwo ? 2 : 1;
        const int ch = units <= 32 ? 1 : units <= 64 ? 2 : ctas == 1 ? (units <= 1024 ? 1 : 4) : units > 512 && units <= 896 ? 2 : 4;
        const int threads = std::max(32, ((units + ch - 1) / ch + 31) / 32 * 32);
        if (ch == 4) ctas = std::min(ctas, 512 / threads);  // 128 registers a thread
        else if (threads > 32) ctas = std::min(ctas, 2);
        const int stages = 2;
        int sms = 0;
        const cudaError_t e = ops_device(&sms, [] {
            cudaError_t e = cudaSuccess;
            for (int set = kTypesAny; set <= kTypesF32F16; ++set)
                for (int ch : {1, 2, 4})
                    for (int threads : {32, 352, 448, 512})
                        if (e == cudaSuccess)
                            e = cudaFuncSetAttribute(rows_kernel(set, ch, threads),
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem);
            return e;
        });
        if (e != cudaSuccess) return e;
        return ops_launch(rows_kernel(set, ch, threads), (unsigned)std::min<int64_t>(tokens, (int64_t)sms * ctas), threads,
                          (size_t)stages * stage, s, a, tokens, stages, y_bytes, h_bytes, g_bytes);
    }
    // Many short rows: a warp each, eight to a CTA (8192 CTAs take 9 us to start). 8192 x 64 bf16 with a
    // channel gate 5.9 for 9.2 us, 8192 x 256 6.1 for 9.2, 2000 x 256 3.1 for 3.5, 600 x 256 2.7 either way;
    // 2000 x 512 unaligned would take 6.4 for 5.1 us.
    if (units <= 32 && tokens >= 1000)
        return ops_launch(row_kernel(set, 0, width), (unsigned)(((int64_t)tokens + 7) / 8), dim3(32, 8), 0, s, a);
    const int ch = units <= 1024 ? 1 : units <= 2048 ? 2 : 4;
    const int threads = std::max(32, ((units + ch - 1) / ch + 31) / 32 * 32);
    return ops_launch(row_kernel(set, ch, width), (unsigned)tokens, threads, 0, s, a);
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
        // the widest accesses that every tensor's alignment allows
        int width = c.dim % 8 == 0 ? 8 : 4;
        auto narrow = [&](const void* p, int type, int64_t ld) {
            while (width > 1 && (!clb::ops_aligned(p, width * clb::ops_type_bytes(type)) || ld % width)) width /= 2;
        };
        for (const Tensor& t : rows) {
            if (!t.p) continue;
            const size_t b = clb::ops_type_bytes(t.type);
            require(t.ld >= c.dim && t.ld <= (int64_t)1 << 40, CLB_E_INVALID, "row pitch of %s below dim", t.name);
            require(clb::ops_aligned(t.p, b), CLB_E_INVALID, "%s is misaligned", t.name);
            narrow(t.p, t.type, t.ld);
        }
        for (const Tensor& t : vecs) {
            if (!t.p) continue;
            require(clb::ops_aligned(t.p, clb::ops_type_bytes(t.type)), CLB_E_INVALID, "%s is misaligned", t.name);
            // a gate for each token is read one number at a time
            if (t.p != d_gate || c.gate == CLB_GATE_CHANNEL) narrow(t.p, t.type, 0);
        }
        // an output over an input: only h_out in h's place, row by row
        const int64_t gate_count = c.gate == CLB_GATE_TOKEN ? tokens : c.dim;
        const clb::OpsRows all[] = {clb::ops_rows("h", d_h, tokens, c.dim, c.ld_h, c.h_type),
                                    clb::ops_rows("y", d_y, tokens, c.dim, c.ld_y, c.y_type),
                                    full ? clb::ops_rows("gate", d_gate, tokens, c.dim, c.ld_gate, c.gate_type)
                                         : clb::ops_rows("gate", d_gate, 1, gate_count, gate_count, c.gate_type),
                                    clb::ops_rows("w_post", d_w_post, 1, c.dim, c.dim, CLB_F32),
                                    clb::ops_rows("w_pre", d_w_pre, 1, c.dim, c.dim, CLB_F32)};
        const clb::OpsRows h_out = clb::ops_rows("h_out", d_h_out, tokens, c.dim, c.ld_h_out, c.h_type);
        const clb::OpsRows x = clb::ops_rows("x", d_x, tokens, c.dim, c.ld_x, c.x_type), to_x[] = {x};
        const bool in_place = d_h_out == d_h && (c.ld_h_out == c.ld_h || tokens == 1);
        for (const clb::OpsRows& t : all)
            require((&t == all && in_place) || clb::ops_apart(h_out, t), CLB_E_INVALID, "h_out overlaps %s", t.name);
        clb::ops_require_apart(x, all);
        clb::ops_require_apart(h_out, to_x);
        clb::NormArgs a{};
        a.h = d_h, a.y = d_y, a.gate = d_gate, a.w_post = d_w_post, a.w_pre = d_w_pre, a.h_out = d_h_out, a.x = d_x;
        a.ld_h = c.ld_h, a.ld_y = c.ld_y, a.ld_gate = c.ld_gate, a.ld_h_out = c.ld_h_out, a.ld_x = c.ld_x;
        a.tokens = tokens, a.dim = c.dim, a.h_type = c.h_type, a.y_type = c.y_type, a.gate_type = c.gate_type, a.x_type = c.x_type;
        a.gate_kind = d_gate ? c.gate : CLB_GATE_NONE, a.gate_sigmoid = c.gate_sigmoid, a.post = c.post;
        a.post_eps = c.post_eps, a.pre_eps = c.pre_eps, a.residual_scale = c.residual_scale;
        a.block_scale = c.block_scale, a.inv_dim = 1.0f / (float)c.dim;
        cuda_check(clb::launch_block_norm(a, tokens, width, static_cast<cudaStream_t>(stream)),
                   "block norm");
    });
}
