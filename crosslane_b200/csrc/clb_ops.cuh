// Helpers shared by the operators around the routed experts (clb_route.cu, clb_block_norm.cu,
// clb_int8.cu): element types, warp reductions, argument checks, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "clb_host.h"

namespace clb {

inline bool ops_float_type(int t) { return t == CLB_F32 || t == CLB_BF16 || t == CLB_F16; }
inline int ops_type_bytes(int t) { return t == CLB_F32 ? 4 : t == CLB_I8 ? 1 : 2; }
inline bool ops_aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// One element of a floating tensor; `type` is uniform over the grid.
__device__ __forceinline__ float ops_load(const void* p, int type, int64_t i) {
    if (type == CLB_F32) return static_cast<const float*>(p)[i];
    const uint16_t b = static_cast<const uint16_t*>(p)[i];
    return type == CLB_BF16 ? __uint_as_float((uint32_t)b << 16) : __half2float(__ushort_as_half(b));
}
__device__ __forceinline__ void ops_store(void* p, int type, int64_t i, float v) {
    if (type == CLB_F32) static_cast<float*>(p)[i] = v;
    else if (type == CLB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Eight elements from i on, 16-byte aligned (coherent loads: the tensor may be updated in place).
__device__ __forceinline__ void load8_aligned(const void* p, int type, int64_t i, float (&v)[8]) {
    if (type == CLB_F32) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return;
    }
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (type == CLB_BF16) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
    }
}

__device__ __forceinline__ float ops_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Launch through cudaLaunchKernelEx, whose own status is the launch's (cudaGetLastError would
// also hand over, and clear, an earlier error of the caller's).
template <class... P, class... A>
cudaError_t ops_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

}  // namespace clb
