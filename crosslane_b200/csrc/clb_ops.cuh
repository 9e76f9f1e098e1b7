// Helpers shared by the operators around the routed experts (clb_route.cu, clb_block_norm.cu,
// clb_int8.cu): element types, warp reductions, argument checks, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "clb_host.h"

namespace clb {

inline bool ops_float_type(int t) { return t == CLB_F32 || t == CLB_BF16 || t == CLB_F16; }
inline int ops_type_bytes(int t) { return t == CLB_F32 ? 4 : t == CLB_I8 ? 1 : 2; }
inline bool ops_aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether eight elements from a multiple of 8 on can be moved at once in every row (32 bytes of
// fp32, 16 of the others).
inline bool ops_vec8(const void* p, int type, int64_t ld) { return ops_aligned(p, type == CLB_F32 ? 32 : 16) && ld % 8 == 0; }

// A tensor's rows in bytes (a vector: one row); an absent tensor holds none.
struct OpsRows {
    const char* name;
    uint64_t lo, hi;  // the first byte and the one behind the last
    int64_t rows, width, pitch;
};
inline OpsRows ops_rows(const char* name, const void* p, int64_t rows, int64_t width, int64_t ld, int type) {
    if (!p || rows < 1) return {name, 0, 0, 0, 0, 0};
    const uint64_t lo = reinterpret_cast<uintptr_t>(p);
    const int b = ops_type_bytes(type);
    const unsigned __int128 hi = lo + ((unsigned __int128)(rows - 1) * (uint64_t)ld + (uint64_t)width) * b;
    return {name, lo, hi >> 64 ? UINT64_MAX : (uint64_t)hi, rows, width * b, ld < ((int64_t)1 << 60) ? ld * b : INT64_MAX};
}
// Whether no row of one shares a byte with a row of the other: apart as ranges, or of one pitch in
// columns apart (rows of one wider buffer interleave).
inline bool ops_apart(const OpsRows& a, const OpsRows& b) {
    if (a.hi <= b.lo || b.hi <= a.lo) return true;
    if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch)) return false;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    const int64_t apart = (int64_t)(a.lo >= b.lo ? a.lo - b.lo : b.lo - a.lo) % pitch;
    const int64_t d = a.lo >= b.lo || apart == 0 ? apart : pitch - apart;  // column of a in b's rows
    return d >= b.width && a.width <= pitch - d;
}
// Refuses an output that lies over one of the others.
template <size_t N>
void ops_require_apart(const OpsRows& out, const OpsRows (&others)[N]) {
    for (const OpsRows& t : others) require(ops_apart(out, t), CLB_E_INVALID, "%s overlaps %s", out.name, t.name);
}

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

// Eight elements as they lie in memory. Loading and converting are two steps, so that a thread
// has all its loads in flight before it touches the first: the element type is a value of the
// launch, and a conversion right behind each load would wait for it.
struct Raw8 {
    uint4 a, b;  // 16-bit types, aligned: in a; otherwise one element a word
};
// The loads are predicated, not branched around, and coherent: the tensor may be updated in place.
__device__ __forceinline__ void ld16_if(uint4& v, const void* p, bool ok) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
                 : "l"(p), "r"((uint32_t)ok));
}
__device__ __forceinline__ void ld32_if(uint4& a, uint4& b, const void* p, bool ok) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %9, 0;\n\t"
        "@p ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t}"
        : "+r"(a.x), "+r"(a.y), "+r"(a.z), "+r"(a.w), "+r"(b.x), "+r"(b.y), "+r"(b.z), "+r"(b.w)
        : "l"(p), "r"((uint32_t)ok));
}
__device__ __forceinline__ void ld_elem_if(uint32_t& v, const void* row, int type, int64_t i, bool ok) {
    const char* p = static_cast<const char*>(row) + i * (type == CLB_F32 ? 4 : 2);
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u16 h;\n\tsetp.ne.u32 p, %2, 0;\n\tsetp.ne.u32 q, %3, 0;\n\t"
        "@p ld.global.u32 %0, [%1];\n\t@q ld.global.u16 h, [%1];\n\t@q cvt.u32.u16 %0, h;\n\t}"
        : "+r"(v)
        : "l"(p), "r"((uint32_t)(ok && type == CLB_F32)), "r"((uint32_t)(ok && type != CLB_F32)));
}
__device__ __forceinline__ void ld4_if(uint32_t& a, const void* p, bool ok) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.global.u32 %0, [%1];\n\t}" : "+r"(a) : "l"(p), "r"((uint32_t)ok));
}
__device__ __forceinline__ void ld8_if(uint32_t& a, uint32_t& b, const void* p, bool ok) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t@p ld.global.v2.u32 {%0, %1}, [%2];\n\t}"
                 : "+r"(a), "+r"(b)
                 : "l"(p), "r"((uint32_t)ok));
}
__device__ __forceinline__ float elem_float(uint32_t v, int type) {
    return type == CLB_F32    ? __uint_as_float(v)
           : type == CLB_BF16 ? __uint_as_float(v << 16)
                              : __half2float(__ushort_as_half((uint16_t)v));
}
// Aligned (ops_vec8): elements i .. i + 7 of `row`, where ok; zeros otherwise.
__device__ __forceinline__ Raw8 raw8_aligned(const void* row, int type, int64_t i, bool ok) {
    Raw8 r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    const char* p = static_cast<const char*>(row) + i * (type == CLB_F32 ? 4 : 2);
    ld32_if(r.a, r.b, p, ok && type == CLB_F32);
    ld16_if(r.a, p, ok && type != CLB_F32);
    return r;
}
// Any alignment: elements i + j * step for the j with i + j * step < n; zeros otherwise.
__device__ __forceinline__ Raw8 raw8_strided(const void* row, int type, int64_t i, int step, int n) {
    Raw8 r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    ld_elem_if(r.a.x, row, type, i, i < n);
    ld_elem_if(r.a.y, row, type, i + step, i + step < n);
    ld_elem_if(r.a.z, row, type, i + 2 * step, i + 2 * step < n);
    ld_elem_if(r.a.w, row, type, i + 3 * step, i + 3 * step < n);
    ld_elem_if(r.b.x, row, type, i + 4 * step, i + 4 * step < n);
    ld_elem_if(r.b.y, row, type, i + 5 * step, i + 5 * step < n);
    ld_elem_if(r.b.z, row, type, i + 6 * step, i + 6 * step < n);
    ld_elem_if(r.b.w, row, type, i + 7 * step, i + 7 * step < n);
    return r;
}
// `packed`: from raw8_aligned.
__device__ __forceinline__ void raw8_floats(const Raw8& r, int type, bool packed, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == CLB_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else if (type == CLB_BF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __uint_as_float(!packed || !(j & 1) ? w[packed ? j / 2 : j] << 16 : w[j / 2] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t pair = packed ? w[j / 2] : w[j] | w[j + 1] << 16;
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
            v[j] = f.x, v[j + 1] = f.y;
        }
    }
}

// Two floats in a register pair: sm_100a multiplies and adds both in one instruction, each rounded
// as the scalar operation is.
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 f2_floats(F2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

// Eight values as four pairs of a 16-bit type.
__device__ __forceinline__ uint4 pack8(int type, const float (&v)[8]) {
    uint32_t w[4];
    if (type == CLB_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 b = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Eight elements from i on, aligned as for raw8_aligned.
__device__ __forceinline__ void store8_aligned(void* p, int type, int64_t i, const float (&v)[8]) {
    if (type == CLB_F32) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<float*>(p) + i), "f"(v[0]),
                     "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
        return;
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = pack8(type, v);
}

// Rows that start anywhere, through shared memory: byte j of the row lies at `smem` + (address mod 16)
// + j, so its whole 16-byte pieces are copied as such (asynchronously: row_landed comes before the
// first use), and the up to 15 bytes on either side by elements. bytes + 48 of shared memory.
__device__ __forceinline__ void row_to_smem(uint32_t smem, const void* row, uint32_t bytes, int type) {
    const char* p = static_cast<const char*>(row);
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u, es = type == CLB_F32 ? 4u : 2u;
    const uint32_t head = min((16u - off) & 15u, bytes), pieces = (bytes - head) >> 4, done = head + 16u * pieces;
    for (uint32_t i = threadIdx.x; i < pieces; i += blockDim.x)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem + off + head + 16u * i), "l"(p + head + 16u * i)
                     : "memory");
    const uint32_t edge = (head + bytes - done) / es;  // elements in front of and behind the pieces
    if (threadIdx.x < edge) {
        const uint32_t at = threadIdx.x * es < head ? threadIdx.x * es : done + threadIdx.x * es - head;
        if (type == CLB_F32)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem + off + at), "l"(p + at) : "memory");
        else
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(smem + off + at), "h"(*reinterpret_cast<const uint16_t*>(p + at))
                         : "memory");
    }
}
__device__ __forceinline__ void row_landed() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}
// Eight elements of such a row from its chunk c on, as raw8_aligned gives them; off: address mod 16.
// The words are moved by selects: a branch for each shift is 8 times the code, and what a launch of
// few rows waits for is its code.
__device__ __forceinline__ Raw8 raw8_smem(uint32_t smem, uint32_t off, int type, int c) {
    uint32_t w[12];
    const uint32_t p = smem + (uint32_t)c * (type == CLB_F32 ? 32u : 16u);
    const int n = type == CLB_F32 ? 8 : 4;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < 2 || type == CLB_F32)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                         : "r"(p + 16u * i));
        else
            w[8] = w[9] = w[10] = w[11] = 0u;
    const bool two = off & 8u, one = off & 4u;
#pragma unroll
    for (int j = 0; j < 10; ++j) w[j] = two ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 9; ++j) w[j] = one ? w[j + 1] : w[j];
    if (n == 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], (off & 2u) << 3);
    return Raw8{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}
__device__ __forceinline__ float ops_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// SMs of the current device; `setup` (kernel attributes) runs once per device and call site.
template <class Setup>
cudaError_t ops_device(int* sms, Setup setup) {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];  // 0: not set up yet
    static std::mutex mutex;
    int dev = 0;
    cudaError_t e;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if (dev < 0 || dev >= kDevices) return cudaErrorInvalidDevice;
    if ((*sms = known[dev].load(std::memory_order_acquire)) > 0) return cudaSuccess;
    std::lock_guard<std::mutex> lock(mutex);
    int count = 0;
    if ((e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = setup()) != cudaSuccess) return e;
    known[dev].store(*sms = count, std::memory_order_release);
    return cudaSuccess;
}

// Launch through cudaLaunchKernelEx, whose own status is the launch's (cudaGetLastError would
// also hand over, and clear, an earlier error of the caller's). The kernel's CTAs may be set
// up while the kernel in front of it on the stream ends: it starts with ops_wait.
template <class... P, class... A>
cudaError_t ops_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = s;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

// The first thing every thread of such a kernel does: waits until all work in front of it on the
// stream has completed and is visible.
// Behind it memory is read by coherent loads alone: the read-only path (ld.global.nc) is for data that
// nobody writes while the kernel runs, and the kernel in front may still be writing when this one's CTAs
// start; such a load may also be moved in front of the wait.
__device__ __forceinline__ void ops_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The same, and lets the kernel behind it be set up under this one. In this order a kernel that runs
// ahead of its own wait knows that all but the one in front is complete.
__device__ __forceinline__ void ops_begin() {
    ops_wait();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace clb
