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
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the product's CTAs may start loading weights
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

// ------------------------------------------------------------------------------
// Tensor-core product: D[128 weight rows][nt tokens] in tensor memory (int32), A = weights
// and B = quantised tokens by TMA (128-byte rows of K, 128-byte swizzle), four
// tcgen05.mma kind::i8 of K = 32 per 128-byte block. Warps 0-3 are the epilogue (a lane is a
// weight row, so a warp's store of one token is contiguous), warp 4 loads, warp 5 issues.
// SPLIT: the CTAs of a cluster share a tile's K range; their sums are added over
// distributed shared memory (integers: the order does not matter). Otherwise a CTA walks
// over tiles, the epilogue of one under the products of the next (two accumulators).
constexpr int kGmThreads = 192;
constexpr int kGmMaxStages = 12;
constexpr int kGmABytes = 128 * 128;
constexpr int kGmSmem = 220 * 1024;           // dynamic shared memory, alignment included
constexpr uint32_t kGmTmemCols = 512, kGmAccCols = 256;
constexpr uint64_t kGmTimeoutNs = 1000000000; // a pipeline wait longer than this is an error
constexpr uint32_t kGmDrainPolls = 1u << 22;

struct Int8Gemm {
    CUtensorMap wmap, xmap;  // [n][k] box 128 rows, [tokens][k] box nt rows; 128 bytes wide
    const float *w_scale, *q_scale, *bias;
    void* out;
    int* status;
    int64_t ld_out;
    int tokens, n, kblocks, nt, stages, mtiles, tiles, split, out_type;
};

// D (+)= A . B^T, both operands described in shared memory.
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// K-major operand, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61) |
           (uint64_t)((addr >> 4) & 0x3FFFu);
}
__device__ __noinline__ bool gm_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
    const uint64_t t0 = tc_now_ns();
    for (;;) {
        if (mbar_try_sleep(bar, parity)) return true;
        if (*abort_flag) return false;
        if (tc_now_ns() - t0 > kGmTimeoutNs) break;
    }
    if (status) atomicExch(status, kErrInt8Wait);
    *abort_flag = 1;
    return false;
}
__device__ __forceinline__ bool gm_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
    return mbar_try(bar, parity) || gm_wait_slow(bar, parity, abort_flag, status);
}

template <bool SPLIT>
__global__ void __launch_bounds__(kGmThreads, 1) k_int8_gemm(const __grid_constant__ Int8Gemm g) {
    extern __shared__ uint8_t gm_smem[];
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
    const uint32_t stage_bytes = (uint32_t)kGmABytes + (uint32_t)g.nt * 128u;
    const int rank = SPLIT ? (int)blockIdx.x % g.split : 0;
    const int first = SPLIT ? (int)blockIdx.x / g.split : (int)blockIdx.x, step = (int)gridDim.x;
    const int my_tiles = SPLIT ? 1 : (g.tiles - 1 - first) / step + 1;
    const int kb0 = SPLIT ? (int)((int64_t)g.kblocks * rank / g.split) : 0;
    const int nkb = (SPLIT ? (int)((int64_t)g.kblocks * (rank + 1) / g.split) : g.kblocks) - kb0;
    const int64_t total = (int64_t)my_tiles * nkb;

    if (tid == 0) {
        for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(empty(i), 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full(i), 1), mbar_init(acc_empty(i), 4);
        mbar_init(drain, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(&tslot)),
                     "r"(kGmTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tslot);

    if (warp == 4) {
        if (lane == 0) {
            // weights do not depend on the quantising kernel in front: their first loads go out before
            // that kernel has finished, the tokens' after
            const int ahead = (int)min((int64_t)g.stages, total);
            int tile = first, kb = 0;
            auto at = [&](int& m, int& t) {
                m = (tile % g.mtiles) * 128;
                t = (tile / g.mtiles) * g.nt;
            };
            for (int i = 0; i < ahead; ++i) {
                int m, t;
                at(m, t);
                mbar_expect_tx(full(i), stage_bytes);
                tma_2d(base + (uint32_t)i * stage_bytes, &g.wmap, (kb0 + kb) * 128, m, full(i));
                if (++kb == nkb) kb = 0, tile += step;
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            tile = first, kb = 0;
            int stage = 0;
            uint32_t phase = 0;
            for (int64_t i = 0; i < total; ++i) {
                int m, t;
                at(m, t);
                const uint32_t a = base + (uint32_t)stage * stage_bytes;
                if (i >= ahead) {
                    if (!gm_wait(empty(stage), phase ^ 1u, abort_flag, g.status)) break;
                    mbar_expect_tx(full(stage), stage_bytes);
                    tma_2d(a, &g.wmap, (kb0 + kb) * 128, m, full(stage));
                }
                tma_2d(a + kGmABytes, &g.xmap, (kb0 + kb) * 128, t, full(stage));
                if (++stage == g.stages) stage = 0, phase ^= 1u;
                if (++kb == nkb) kb = 0, tile += step;
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            // D s32, A and B signed 8-bit, N and M of the instruction
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(g.nt >> 3) << 17) | (8u << 24);
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
                        umma_i8(tmem + (uint32_t)acc * kGmAccCols, da + 2u * j, db + 2u * j, idesc, kb > 0 || j > 0);
                    umma_commit(empty(stage));
                    if (++stage == g.stages) stage = 0, phase ^= 1u;
                }
                if (ok) umma_commit(acc_full(acc));
            }
        }
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // q_scale
        const uint32_t tlane = tmem + ((uint32_t)(32 * warp) << 16);
        bool ok = true;
        for (int i = 0; i < my_tiles && ok; ++i) {
            const int acc = i & 1, tile = first + i * step;
            const int row = (tile % g.mtiles) * 128 + tid, t0 = (tile / g.mtiles) * g.nt;
            ok = __all_sync(0xffffffffu, gm_wait(acc_full(acc), (uint32_t)(i >> 1) & 1u, abort_flag, g.status));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float ws = row < g.n ? g.w_scale[row] : 0.0f;
            const float bias = g.bias && row < g.n ? g.bias[row] : 0.0f;
            for (int c = 0; c < g.nt; c += 16) {
                int r[16];
                tmem_ld16(tlane + (uint32_t)acc * kGmAccCols + (uint32_t)c, r);
                const int mine = t0 + c + (lane & 15);
                const float xs = !SPLIT && mine < g.tokens ? g.q_scale[mine] : 0.0f;
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (SPLIT) {  // the sums of this K range, [token][row]; every product has completed, so the
                                  // stages are free
                        asm volatile("st.shared.s32 [%0], %1;" ::"r"(base + (uint32_t)((c + j) * 128 + tid) * 4u), "r"(r[j]));
                    } else {
                        const float x = __shfl_sync(0xffffffffu, xs, j);
                        if (row < g.n && t0 + c + j < g.tokens)
                            ops_store(g.out, g.out_type, (t0 + c + j) * g.ld_out + row,
                                      int8_value(r[j], x, ws, bias, g.bias != nullptr));
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(acc));
        }
    }

    if (SPLIT) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        const int row = (first % g.mtiles) * 128 + tid, t0 = (first / g.mtiles) * g.nt;
        if (tid < 128 && row < g.n) {
            const float ws = g.w_scale[row], bias = g.bias ? g.bias[row] : 0.0f;
            for (int c = g.nt * rank / g.split; c < g.nt * (rank + 1) / g.split && t0 + c < g.tokens; ++c) {
                int sum = 0;
#pragma unroll 8
                for (int p = 0; p < g.split; ++p) {
                    uint32_t addr;
                    int v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                 : "=r"(addr)
                                 : "r"(base + (uint32_t)(c * 128 + tid) * 4u), "r"(p));
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
                    sum += v;
                }
                ops_store(g.out, g.out_type, (t0 + c) * g.ld_out + row,
                          int8_value(sum, g.q_scale[t0 + c], ws, bias, g.bias != nullptr));
            }
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }
    __syncthreads();
    if (*abort_flag) {  // let copies in flight land and the issued products complete before leaving
        const uint64_t t0 = tc_now_ns();
        while (tc_now_ns() - t0 < 200000u) {
        }
        if (warp == 5 && lane == 0) {
            umma_commit(drain);
            for (uint32_t i = 0; i < kGmDrainPolls && !mbar_try(drain, 0); ++i) {
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kGmTmemCols));
}

// The tile width and the K split of a product, by an estimate of its SM cycles: a 128-byte
// block of K costs the larger of its products (2 cycles a token column at 8192 multiply-adds
// per cycle) and its loads (kGmLoadRate bytes per cycle and SM), a tile a fixed part; the CTAs
// run in waves over the SMs.
constexpr double kGmLoadRate = 48.0, kGmTileCycles = 700.0, kGmSplitCycles = 1500.0;
struct GmPlan {
    int nt, split;
};
GmPlan gm_plan(int tokens, int n, int kblocks, int sms) {
    GmPlan best{16, 1};
    double least = 1e300;
    const int64_t mt = (n + 127) / 128;
    for (int nt = 16; nt <= 256; nt += 16) {
        if (nt > 16 && nt - 16 >= tokens) break;
        const int64_t tiles = mt * ((tokens + nt - 1) / nt);
        for (int split = 1; split <= 8 && split <= kblocks; split *= 2) {
            if (split > 1 && (nt > 128 || tiles * split > sms)) break;
            const int64_t waves = (tiles * split + sms - 1) / sms;
            const double block = std::max(2.0 * nt, (128.0 + nt) * 128.0 / kGmLoadRate);
            const double per = ((kblocks + split - 1) / split) * block + kGmTileCycles + 4.0 * nt;
            const double cost = waves * per + (split > 1 ? kGmSplitCycles : 0.0);
            if (cost < least) least = cost, best = GmPlan{nt, split};
        }
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

cudaError_t launch_int8_gemm(const Int8Args& a, int* status, bool overlap, cudaStream_t s) {
    int dev = 0, sms = 0;
    cudaError_t e;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    Int8Gemm g{};
    g.kblocks = (a.k + 127) / 128;
    const GmPlan plan = gm_plan(a.tokens, a.n, g.kblocks, sms);
    g.nt = plan.nt, g.split = plan.split;
    if ((e = gm_encode(&g.wmap, a.w, a.n, a.k, a.ld_w, 128)) != cudaSuccess) return e;
    if ((e = gm_encode(&g.xmap, a.q, a.tokens, a.k, a.ld_q, g.nt)) != cudaSuccess) return e;
    g.w_scale = a.w_scale, g.q_scale = a.q_scale, g.bias = a.bias, g.out = a.out, g.status = status;
    g.ld_out = a.ld_out, g.tokens = a.tokens, g.n = a.n, g.out_type = a.out_type;
    g.stages = std::min(kGmMaxStages, (kGmSmem - 1024) / (kGmABytes + g.nt * 128));
    g.mtiles = (a.n + 127) / 128;
    g.tiles = g.mtiles * ((a.tokens + g.nt - 1) / g.nt);
    void (*kernel)(Int8Gemm) = g.split > 1 ? k_int8_gemm<true> : k_int8_gemm<false>;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGmSmem)) != cudaSuccess) return e;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(g.split > 1 ? g.tiles * g.split : std::min(g.tiles, sms)));
    c.blockDim = dim3(kGmThreads);
    c.dynamicSmemBytes = kGmSmem;
    c.stream = s;
    c.attrs = attr;
    if (g.split > 1) {
        attr[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[c.numAttrs].val.clusterDim.x = (unsigned)g.split;
        attr[c.numAttrs].val.clusterDim.y = attr[c.numAttrs].val.clusterDim.z = 1;
        ++c.numAttrs;
    }
    if (overlap) {
        attr[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++c.numAttrs;
    }
    return cudaLaunchKernelEx(&c, kernel, g);
}

// Up to this many tokens the product is row dots, above it tensor-core tiles.
constexpr int kDotTokens = 8;

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
        if (tokens > clb::kDotTokens) {
            cuda_check(clb::launch_int8_gemm(a, d_status, !ready, s), "int8 product");
            return;
        }
        cuda_check(clb::ops_launch(clb::k_int8_dot, dim3((unsigned)((c.n + 7) / 8), (unsigned)((tokens + 7) / 8)), 256,
                                   0, s, a),
                   "int8 product");
    });
}
