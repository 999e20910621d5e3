// serving_common.cuh -- pieces shared by the serving operators (kv_cache.cu,
// kv_attention.cu, lora.cu).  Internal header.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "hxq_cuda.h"
#include "hxq_serving.h"

namespace hxq {

// Adds to hxq_cuda_launch_count (hxq_cuda_rt.cu).
void count_launches(unsigned n);

namespace serving {

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// One code as the value it stands for (before its scale).
template <int FMT> __device__ __forceinline__ float code_value(uint8_t c)
{
    if (FMT == HXQ_KV_INT8) return (float)(int8_t)c;
    __nv_fp8_e4m3 v;
    v.__x = c;
    return (float)v;
}

// The nearest code (ties to even); int8 takes NaN to 0.
template <int FMT> __device__ __forceinline__ uint8_t nearest_code(float v)
{
    if (FMT == HXQ_KV_INT8) return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));
    return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ void flag(uint32_t *status, uint32_t bit)
{
    if (status) atomicOr(status, bit);
}

// Programmatic dependent launch: the next kernel of the stream may begin its
// prologue / this kernel's reads of its predecessor's results may begin.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

inline hxq_error_t launched(unsigned n = 1)
{
    if (cudaGetLastError() != cudaSuccess) return HXQ_ERR_CUDA;
    count_launches(n);
    return HXQ_OK;
}

inline int sm_count()
{
    static std::atomic<int> known[64];   // by device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 148;
    }
    int sms = known[dev].load(std::memory_order_relaxed);
    if (sms == 0) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
            cudaGetLastError();
            return 148;
        }
        known[dev].store(sms, std::memory_order_relaxed);
    }
    return sms;
}

// Raise a kernel's dynamic shared memory limit, once per device (`ready`:
// one bit per device, a static of the kernel's launcher).
template <typename K> cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<uint64_t> &ready)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (ready.load(std::memory_order_acquire) >> dev & 1u) return cudaSuccess;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)) != cudaSuccess) return e;
    ready.fetch_or(1ull << dev, std::memory_order_acq_rel);
    return cudaSuccess;
}

// A launch that may begin before the kernel in front of it on the stream
// has ended; the kernel calls wait_previous before it reads or writes memory.
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Host side: runs of `width` consecutive elements, n[0] x n[1] of them,
// stride[] elements apart.
struct Runs {
    uintptr_t at;
    int64_t n[2], stride[2];
    int64_t width, size;   // elements of a run, bytes of an element

    static __int128 far(__int128 v) { return v < 0 ? -v : v; }
    bool longer0() const { return n[1] == 1 || (n[0] > 1 && far(stride[0]) >= far(stride[1])); }

    // Whether every element has its own place, one stride being beyond all that
    // the other one spans.
    bool apart() const
    {
        const int o = longer0() ? 0 : 1, i = 1 - o;
        const __int128 inner = n[i] > 1 ? (n[i] - 1) * far(stride[i]) + width : width;
        return (n[i] == 1 || far(stride[i]) >= width) && (n[o] == 1 || far(stride[o]) >= inner);
    }
    void range(__int128 &lo, __int128 &hi) const
    {
        lo = hi = (__int128)at;
        for (int d = 0; d < 2; ++d) ((stride[d] < 0) ? lo : hi) += (__int128)(n[d] - 1) * stride[d] * size;
        hi += (__int128)width * size;
    }
    // Whether a call may write these (which are apart) and read the others: if
    // they are the same elements in the same places, or share none. Where the
    // strides differ that is told by the ranges alone.
    bool may_overwrite(const Runs &r) const
    {
        __int128 a0, a1, b0, b1;
        range(a0, a1);
        r.range(b0, b1);
        if (a1 <= b0 || b1 <= a0) return true;
        for (int d = 0; d < 2; ++d)
            if (n[d] > 1 && stride[d] != r.stride[d]) return false;
        const __int128 bytes = (__int128)at - (__int128)r.at;
        if (bytes == 0) return true;
        if (bytes % size) return false;
        const int o = longer0() ? 0 : 1, i = 1 - o;
        auto below = [](__int128 v, __int128 by) { return v >= 0 ? v / by : -((-v + by - 1) / by); };
        const __int128 so = n[o] > 1 ? stride[o] : 1, si = n[i] > 1 ? stride[i] : 1, delta = bytes / size;
        for (int u = 0; u < 2; ++u)
            for (int v = 0; v < 2; ++v) {
                const __int128 x = n[o] > 1 ? below(delta, far(so)) + u : 0, rest = delta - x * far(so);
                const __int128 y = n[i] > 1 ? below(rest, far(si)) + v : 0;
                if (far(x) < n[o] && far(y) < n[i] && far(rest - y * far(si)) < width) return false;
            }
        return true;
    }
};

// Host checks of a cache descriptor.
inline hxq_error_t check_cache(const hxq_kv_cache_t *c)
{
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales) return HXQ_ERR_NULL_PTR;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return HXQ_ERR_INVALID_DIM;
    if (c->block_tokens == 0 || c->block_tokens % 16 != 0 || c->block_tokens > 256) return HXQ_ERR_INVALID_DIM;
    if (c->n_blocks == 0 || c->n_heads == 0 || c->n_heads > 65535) return HXQ_ERR_INVALID_ARG;
    if ((uint64_t)c->n_blocks * c->block_tokens >= (1ull << 31)) return HXQ_ERR_INVALID_ARG;
    if (c->format != HXQ_KV_INT8 && c->format != HXQ_KV_E4M3) return HXQ_ERR_INVALID_ARG;
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15u) != 0 || (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 3u) != 0)
        return HXQ_ERR_INVALID_ARG;
    return HXQ_OK;
}

}  // namespace serving
}  // namespace hxq
