// sm100.cuh — device and host helpers shared by the decoder-layer operators
// (norm.cu, linear.cu, kv4.cu).  Not part of the C ABI.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "../../include/tans_b200.h"
#include "internal.h"

namespace tans_b200 {

// ------------------------------------------------- programmatic launch
//
// Every kernel of these operators is launched so that it may start while the
// kernel before it on the stream drains, and touches global memory only after
// pdl_wait(), when that kernel is complete and its writes are visible.  It
// lets the next kernel in only after its own wait, so whatever that one reads
// early (the GEMV's weight) was written by a kernel already complete.
__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

inline int launch_failed(const char *name, cudaError_t e) {
    (void)cudaGetLastError();
    return fail(TANS_B200_ERR_CUDA, "%s launch: %s", name, cudaGetErrorString(e));
}

// `cluster` > 1: CTAs of a cluster are consecutive in x.
template <typename... P, typename... A>
int launch_ex(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st,
              const char *name, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
    return e == cudaSuccess ? TANS_B200_OK : launch_failed(name, e);
}

constexpr int kMaxDevices = 64;

// The current device and its SM count (asked for once per device).
inline int current_sms(const char *what, int *sms) {
    static std::atomic<int> known[kMaxDevices];
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) e = cudaErrorInvalidDevice;
    if (e != cudaSuccess) return launch_failed(what, e);
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return launch_failed(what, e);
        known[dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return TANS_B200_OK;
}

// Lets `kernel` use up to `bytes` of dynamic shared memory on the current
// device, which has to be the same for every call: done once per device.
template <auto kernel>
int allow_smem(const char *what, int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) e = cudaErrorInvalidDevice;
    if (e != cudaSuccess) return launch_failed(what, e);
    if (done.load(std::memory_order_relaxed) >> dev & 1) return TANS_B200_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return launch_failed(what, e);
    done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return TANS_B200_OK;
}

inline bool is_aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
// whether elements of `size` bytes may lie at each of p (null: yes)
template <typename... P>
bool may_hold(uintptr_t size, const P *...p) {
    return (is_aligned(p, size) && ...);
}
inline uintptr_t element_bytes(int dtype) { return dtype == TANS_B200_F32 ? 4 : 2; }

template <typename I>
__host__ __device__ constexpr I ceil_div(I a, I b) {
    return (a + b - 1) / b;
}

// ------------------------------------------------------------ element types

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same_v<T, float>)
        return v;
    else if constexpr (std::is_same_v<T, __half>)
        return __half2float(v);
    else
        return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (std::is_same_v<T, float>)
        return v;
    else if constexpr (std::is_same_v<T, __half>)
        return __float2half_rn(v);
    else
        return __float2bfloat16_rn(v);
}

// Eight consecutive values, 16-byte aligned (32 for float).
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 u;
        T *e = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint4 *>(p) = u;
    }
}

// Eight consecutive values as they lie in memory, 16-byte aligned.
template <typename T>
struct Eight {
    uint4 u[sizeof(T) / 2];
    __device__ __forceinline__ void to(float (&v)[8]) const {
        const T *e = reinterpret_cast<const T *>(u);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
    }
};
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *p) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.u[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}

// Two e4m3 bytes (low byte = lo), round to nearest even, clamped to +-448;
// NaN becomes 0x7F.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// f(T{}) for the element type of a TANS_B200_BF16 / F16 / F32 code.
template <typename F>
int dispatch_half(int dtype, const char *what, F &&f) {
    if (dtype == TANS_B200_BF16) return f(__nv_bfloat16{});
    if (dtype == TANS_B200_F16) return f(__half{});
    return fail(TANS_B200_ERR_INVALID, "%s: unsupported element type %d", what, dtype);
}
template <typename F>
int dispatch_float(int dtype, const char *what, F &&f) {
    if (dtype == TANS_B200_F32) return f(float{});
    return dispatch_half(dtype, what, std::forward<F>(f));
}

}  // namespace tans_b200
