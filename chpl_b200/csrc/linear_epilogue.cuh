// Activations, their slopes, and the epilogue of the linear-layer products.
#pragma once

#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace linear {

// 1 / (1 + exp(-v)); exp and the reciprocal by the hardware's approximations
// (relative error below 2^-20 where the result matters to 16 bits)
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// act(z).  The tanh form uses 1/2 (1 + tanh u) = sigmoid(2u), which keeps the
// relative accuracy of the left tail.  ReLU passes a NaN on.
template <int ACT>
__device__ __forceinline__ float activate(float z)
{
    if (ACT == CHPL_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (ACT == CHPL_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    if (ACT == CHPL_ACT_GELU_TANH) return z * sigmoid(2.0f * kGeluC * z * (1.0f + kGeluA * z * z));
    if (ACT == CHPL_ACT_SILU) return z * sigmoid(z);
    return z;
}

// act'(z), and act(z) from the same transcendental.  Where the slope has
// settled, |z| above 20, its polynomial factors are held at 20 so that they
// cannot overflow against a zero.
template <int ACT>
__device__ __forceinline__ void slope_and_value(float z, float& slope, float& value)
{
    if (ACT == CHPL_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : 0.0f;
        value = z < 0.0f ? 0.0f : z;
    } else if (ACT == CHPL_ACT_GELU) {
        const float cdf = 0.5f + 0.5f * erff(z * 0.70710678118654752f);
        slope = cdf + z * (0.3989422804014327f * __expf(-0.5f * z * z));
        value = z * cdf;
    } else if (ACT == CHPL_ACT_GELU_TANH) {
        const float s = sigmoid(2.0f * kGeluC * z * (1.0f + kGeluA * z * z));
        const float zc = fminf(fmaxf(z, -20.0f), 20.0f);
        slope = s + zc * (s * (1.0f - s)) * (2.0f * kGeluC * (1.0f + 3.0f * kGeluA * zc * zc));
        value = z * s;
    } else if (ACT == CHPL_ACT_SILU) {
        const float s = sigmoid(z);
        const float zc = fminf(fmaxf(z, -20.0f), 20.0f);
        slope = s * (1.0f + zc * (1.0f - s));
        value = z * s;
    } else {
        slope = 1.0f;
        value = z;
    }
}

// f(std::integral_constant-like tag) with the activation as a compile-time value
template <int V>
struct ActTag {
    static constexpr int value = V;
};

template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f)
{
    switch (act) {
        case CHPL_ACT_RELU: f(ActTag<CHPL_ACT_RELU>()); break;
        case CHPL_ACT_GELU: f(ActTag<CHPL_ACT_GELU>()); break;
        case CHPL_ACT_GELU_TANH: f(ActTag<CHPL_ACT_GELU_TANH>()); break;
        case CHPL_ACT_SILU: f(ActTag<CHPL_ACT_SILU>()); break;
        default: f(ActTag<CHPL_ACT_NONE>()); break;
    }
}

// The epilogue of one thread: its feature f (lane l of a warp holds f0 + l, f0
// a multiple of 32, so a warp holds one checkpoint group) and NB consecutive
// rows t0 .. t0 + NB - 1, D in v.  Every lane of the warp calls it.  Each store
// or load of a row is one coalesced 64-byte (16-bit) access of the warp.
template <typename T, Kind KIND, int NB>
__device__ __forceinline__ void epilogue(const Epilogue& e, int f, int t0, float (&v)[NB], float bias)
{
    const bool ok = f < e.m;
    const int nt = min(NB, e.n - t0);
    if (KIND == kGradWeight) {
        if (!ok) return;
        if (e.out_f32) {
            float* o = static_cast<float*>(e.out) + (int64_t)t0 * e.ldo + f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (j < nt) o[j * e.ldo] = e.accumulate ? o[j * e.ldo] + v[j] : v[j];
        } else {
            T* o = static_cast<T*>(e.out) + (int64_t)t0 * e.ldo + f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (j < nt) o[j * e.ldo] = from_f32<T>(e.accumulate ? to_f32(o[j * e.ldo]) + v[j] : v[j]);
        }
        return;
    }
    // the addend's loads go first, so that they are under way during the arithmetic
    float add[NB];
    if (e.add) {
        const T* a = static_cast<const T*>(e.add) + (int64_t)t0 * e.ldadd + f;
#pragma unroll
        for (int j = 0; j < NB; ++j) add[j] = ok && j < nt ? to_f32(a[j * e.ldadd]) : 0.0f;
    }
    if (KIND == kForward) {
#pragma unroll
        for (int j = 0; j < NB; ++j) v[j] += bias;
        if (e.z && ok) {
            T* o = static_cast<T*>(e.z) + (int64_t)t0 * e.ldz + f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (j < nt) o[j * e.ldz] = from_f32<T>(v[j]);
        }
        if (e.z8.codes) {
            const int g = f / kCkptGroup;
            int8_t* o = e.z8.codes + (int64_t)t0 * e.z8.ldc + f;
            uint8_t* os = e.z8.scales + (int64_t)t0 * e.z8.lds + g;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const uint32_t bits = ok ? __float_as_uint(v[j]) & 0x7fffffffu : 0u;
                const uint32_t s = ckpt_scale(__reduce_max_sync(0xffffffffu, bits));
                const uint32_t code = s == kCkptBadScale ? 0u : ckpt_code(v[j], ckpt_inv_step(s));
                if (ok && j < nt) {
                    o[j * e.z8.ldc] = (int8_t)code;
                    if ((f & (kCkptGroup - 1)) == 0) os[j * e.z8.lds] = (uint8_t)s;
                }
            }
        }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < NB; ++j) v[j] = activate<decltype(tag)::value>(v[j]);
        });
    } else if (e.act != CHPL_ACT_NONE) {
        float z[NB];
        if (e.z8.codes) {
            const int8_t* i = e.z8.codes + (int64_t)t0 * e.z8.ldc + f;
            const uint8_t* is = e.z8.scales + (int64_t)t0 * e.z8.lds + f / kCkptGroup;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                z[j] = ok && j < nt ? (float)i[j * e.z8.ldc] * ckpt_step(is[j * e.z8.lds]) : 0.0f;
        } else {
            const T* i = static_cast<const T*>(e.z) + (int64_t)t0 * e.ldz + f;
#pragma unroll
            for (int j = 0; j < NB; ++j) z[j] = ok && j < nt ? to_f32(i[j * e.ldz]) : 0.0f;
        }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                float slope;
                slope_and_value<decltype(tag)::value>(z[j], slope, z[j]);
                v[j] *= slope;
            }
        });
        if (e.xv && ok) {
            T* o = static_cast<T*>(e.xv) + (int64_t)t0 * e.ldxv + f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (j < nt) o[j * e.ldxv] = from_f32<T>(z[j]);
        }
    }
    if (ok) {
        T* o = static_cast<T*>(e.out) + (int64_t)t0 * e.ldo + f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (j < nt) o[j * e.ldo] = from_f32<T>(e.add ? v[j] + add[j] : v[j]);
    }
}

template <typename T>
__device__ __forceinline__ float bias_of(const Epilogue& e, int f)
{
    return e.bias && f < e.m ? to_f32(static_cast<const T*>(e.bias)[f]) : 0.0f;
}

}  // namespace linear
}  // namespace chpl
