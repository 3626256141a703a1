// Types, activations and reductions that the operators share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "capi_train.h"

namespace stdml::collective::train
{
constexpr int kBf16 = 8, kF16 = 9, kF32 = 10;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v)
{
    return __float2half_rn(v);
}

// Parameters, of which a kernel reads few: their type is looked up at each access.
__device__ __forceinline__ float load_any(const void *p, long long i, int dt)
{
    if (dt == kBf16) { return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]); }
    if (dt == kF16) { return __half2float(static_cast<const __half *>(p)[i]); }
    return static_cast<const float *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, long long i, int dt, float v)
{
    if (dt == kBf16) {
        static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    } else if (dt == kF16) {
        static_cast<__half *>(p)[i] = __float2half_rn(v);
    } else {
        static_cast<float *>(p)[i] = v;
    }
}

// Activations and their derivatives.  `Z`: float, or double where a value next to a
// border is placed.
constexpr float kSqrtHalf = 0.70710678118654752f;   // 1 / sqrt(2)
constexpr float kGauss = 0.39894228040143268f;      // 1 / sqrt(2 pi)
constexpr float kTanhScale = 0.79788456080286536f;  // sqrt(2 / pi)
constexpr float kTanhCube = 0.044715f;

template <int kAct>
__device__ __forceinline__ float act(float z)
{
    if constexpr (kAct == STDMLC_ACT_RELU) { return z > 0.f ? z : (z != z ? z : 0.f); }
    if constexpr (kAct == STDMLC_ACT_SILU) { return z / (1.f + expf(-z)); }
    if constexpr (kAct == STDMLC_ACT_GELU) { return 0.5f * z * (1.f + erff(z * kSqrtHalf)); }
    if constexpr (kAct == STDMLC_ACT_GELU_TANH) {
        return 0.5f * z * (1.f + tanhf(kTanhScale * (z + kTanhCube * z * z * z)));
    }
    return z;
}

template <int kAct>
__device__ __forceinline__ float act_grad(float z)
{
    if constexpr (kAct == STDMLC_ACT_RELU) { return z > 0.f ? 1.f : 0.f; }
    if constexpr (kAct == STDMLC_ACT_SILU) {
        const float s = 1.f / (1.f + expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    if constexpr (kAct == STDMLC_ACT_GELU) {
        return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * kGauss * expf(-0.5f * z * z);
    }
    if constexpr (kAct == STDMLC_ACT_GELU_TANH) {
        const float th = tanhf(kTanhScale * (z + kTanhCube * z * z * z));
        return 0.5f * (1.f + th) +
               0.5f * z * (1.f - th * th) * kTanhScale * (1.f + 3.f * kTanhCube * z * z);
    }
    return 1.f;
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { v += __shfl_xor_sync(0xffffffffu, v, o); }
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o)); }
    return v;
}

// Over all threads of a block (a multiple of 32), in a fixed order; `slots`: 32 values of shared
// memory.  Every thread gets the result.
template <typename V>
__device__ __forceinline__ V block_sum(V v, V *slots)
{
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    __syncthreads();
    if (lane == 0) { slots[warp] = v; }
    __syncthreads();
    return warp_sum(lane < warps ? slots[lane] : V(0));
}
__device__ __forceinline__ float block_max(float v, float *slots)
{
    v = warp_max(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    __syncthreads();
    if (lane == 0) { slots[warp] = v; }
    __syncthreads();
    return warp_max(lane < warps ? slots[lane] : -INFINITY);
}
}  // namespace stdml::collective::train
