// Types, activations and reductions that the operators share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

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

// 16 bytes of T from as many values.  (Two at a time: one alone is converted on the unit of the exponential, at an
// eighth of the rate.)
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half)
{
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float *v)
{
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    } else {
        return make_uint4(pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{}), pack2(v[4], v[5], T{}), pack2(v[6], v[7], T{}));
    }
}
// And back.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &raw, float *v)
{
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
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

constexpr float kSqrtHalf = 0.70710678118654752f;   // 1 / sqrt(2)
constexpr float kGauss = 0.39894228040143268f;      // 1 / sqrt(2 pi)
constexpr float kTanhScale = 0.79788456080286536f;  // sqrt(2 / pi)
constexpr float kTanhCube = 0.044715f;

// The hardware's exponential (base 2) and reciprocal, off by about 2^-22.
__device__ __forceinline__ float fast_exp2(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float fast_rcp(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2E = 1.4426950408889634f;

// z's activation and the derivative there, for results of type T.  32-bit results take CUDA's functions.  For 16-bit
// ones the exponential and the quotient are the hardware's, and erfc(x) = 2 exp(-x^2) poly(1 / (1 + 0.33 x)), whose exponential the
// derivative needs anyway.  The polynomial was fitted to exp(x^2) erfc(x) / 2 for the least maximum of the relative error over x up to 9.5,
// 8.2e-8; with what 32 bits lose, gelu is 4 x 2^-24 |z| off at most, and left of zero 2e-6 of itself down to z = -6 and 8e-6 to -12 (half a
// step of f16 is 2.4e-4 at least).  (The kernels would otherwise spend longer on erf than on memory.)
template <typename T, int kAct>
__device__ __forceinline__ void act_both(float z, float &a, float &d)
{
    constexpr bool kExact = sizeof(T) == 4;
    if constexpr (kAct == STDMLC_ACT_NONE) {
        a = z;
        d = 1.f;
    } else if constexpr (kAct == STDMLC_ACT_RELU) {
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(a) : "f"(z));
        d = z > 0.f ? 1.f : 0.f;
    } else if constexpr (kAct == STDMLC_ACT_SILU) {
        const float s = kExact ? 1.f / (1.f + expf(-z)) : fast_rcp(1.f + fast_exp2(-kLog2E * z));
        a = z * s;
        d = s + a * (1.f - s);
    } else if constexpr (kAct == STDMLC_ACT_GELU && kExact) {
        const float c = 0.5f * (1.f + erff(z * kSqrtHalf));
        a = z * c;
        d = c + z * kGauss * expf(-0.5f * z * z);
    } else if constexpr (kAct == STDMLC_ACT_GELU) {
        // q = erfc(|z| / sqrt 2) / 2: z (1 - q) right of zero, z q left of it.  (Beyond 30, where q is 0, |z| does not
        // matter; an infinity would.)
        const float x = fminf(fabsf(z), 30.f), t = fast_rcp(1.f + 0.33f * kSqrtHalf * x), e = fast_exp2(-0.5f * kLog2E * z * z);
        const float q = e * t * (0.0931830449f + t * (0.0914187618f + t * (0.100961095f + t * (0.022507869f + t * (0.206266189f +
                                 t * (-0.177714604f + t * (0.231341345f - t * 0.0679637408f)))))));
        a = fmaxf(z, 0.f) - x * q;
        d = (z < 0.f ? q : 1.f - q) + z * (kGauss * e);
    } else {
        // s = (1 + tanh y) / 2, which is 0 or 1 long before |z| = 30
        const float z2 = fminf(z * z, 900.f), y = kTanhScale * z * (1.f + kTanhCube * z2);
        const float s = kExact ? 1.f / (1.f + expf(-2.f * y)) : fast_rcp(1.f + fast_exp2(-2.f * kLog2E * y));
        a = z * s;
        d = s + 2.f * a * (1.f - s) * kTanhScale * (1.f + 3.f * kTanhCube * z2);
    }
}
template <typename T, int kAct>
__device__ __forceinline__ float act(float z)
{
    float a, d;
    act_both<T, kAct>(z, a, d);
    return a;
}
template <typename T, int kAct>
__device__ __forceinline__ float act_grad(float z)
{
    float a, d;
    act_both<T, kAct>(z, a, d);
    return d;
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
