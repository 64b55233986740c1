// 8-bit activation checkpoints: the coding of one group, and 16/32-bit element
// conversions shared by the kernels that write or read such checkpoints.
//
// A group of 32 consecutive features shares the step 2^(s - 133), s the FP32
// exponent field of the group's largest magnitude (>= 7), so |x| / step < 128
// and a code is x / step rounded to 7 bits and a sign: code * step is exact in
// bf16, which lets the backward products take a checkpoint as it is.  s >= 7
// keeps step and 1 / step normal FP32 numbers (magnitudes below 2^-126 code to 0).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace chpl {

constexpr int kCkptGroup = 32;
constexpr uint32_t kCkptMinScale = 7;
constexpr uint32_t kCkptBadScale = 255;  // the group held an infinity or a NaN

// scale of a group from the largest FP32 bit pattern (sign cleared) in it; a
// NaN's pattern is above every number's, so a plain integer maximum finds it
__device__ __forceinline__ uint32_t ckpt_scale(uint32_t max_bits)
{
    const uint32_t e = max_bits >> 23;
    return e < kCkptMinScale ? kCkptMinScale : e;
}

// 2^(133 - s); 0 for a poisoned group, whose codes are 0
__device__ __forceinline__ float ckpt_inv_step(uint32_t s)
{
    return s == kCkptBadScale ? 0.0f : __uint_as_float((260u - s) << 23);
}

// 2^(s - 133); NaN for a poisoned group
__device__ __forceinline__ float ckpt_step(uint32_t s)
{
    return s == kCkptBadScale ? __uint_as_float(0x7fffffffu) : __uint_as_float((s - 6u) << 23);
}

// Code of x: x * inv is exact (a power of two, no underflow to speak of: what
// it could lose is below half a code), rounded half to even.  In a poisoned
// group inv is 0, and x * 0 of an infinity or a NaN converts to 0.
__device__ __forceinline__ int ckpt_code(float x, float inv)
{
    const int c = __float2int_rn(x * inv);
    return max(-127, min(127, c));
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace chpl
