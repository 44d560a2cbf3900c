// paged_values.cuh — vectors of 8 values of a row of any of the cache's types, and the
// launch that lets a kernel's start overlap the end of the one before it.
#pragma once

#include "paged.cuh"

namespace kore {
namespace {

struct F8 {
    float v[8];
};

template <typename T>
__device__ __forceinline__ float to_f(T x) {
    return (float)x;
}

template <typename T>
__device__ __forceinline__ F8 load8(const T *p) {
    F8 r;
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
        r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const T *h = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = (float)h[i];
    }
    return r;
}

__device__ __forceinline__ uint16_t two_e4m3(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// scale: of an 8-bit cache (the stored 8 bits are x / scale); 1 otherwise
template <typename T>
__device__ __forceinline__ void store8(T *p, const F8 &x, float scale) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
    } else if constexpr (sizeof(T) == 2) {
        uint4 a;
        T *h = reinterpret_cast<T *>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (T)x.v[i];
        *reinterpret_cast<uint4 *>(p) = a;
    } else {
        uint2 a;
        uint16_t *h = reinterpret_cast<uint16_t *>(&a);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            h[i] = two_e4m3(__fdiv_rn(x.v[2 * i], scale), __fdiv_rn(x.v[2 * i + 1], scale));
        *reinterpret_cast<uint2 *>(p) = a;
    }
}

template <typename T>
__device__ __forceinline__ void store1(T *p, float x, float scale) {
    if constexpr (sizeof(T) == 1)
        *reinterpret_cast<uint8_t *>(p) = (uint8_t)two_e4m3(__fdiv_rn(x, scale), 0.f);
    else
        *p = (T)x;
}

template <typename... Args>
cudaError_t launch(void (*kernel)(Args...), dim3 blocks, int threads, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
}  // namespace kore
