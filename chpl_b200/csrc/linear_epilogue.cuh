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

// Phi(z), the normal distribution function, and E = exp(-z^2 / 2) by the way:
// Abramowitz and Stegun 7.1.26 (Hastings), erfc(x) = t (a1 + ... + a5 t^4) E
// with t = 1 / (1 + p x), x = |z| / sqrt(2), absolute error below 1.5e-7.  One
// exponential and one reciprocal, and the slope's density is E again.
__device__ __forceinline__ float normal_cdf(float z, float& E)
{
    E = __expf(-0.5f * z * z);
    const float t = __fdividef(1.0f, 1.0f + 0.3275911f * 0.70710678f * fabsf(z));
    const float poly = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float tail = 0.5f * poly * E;
    return z < 0.0f ? tail : 1.0f - tail;
}

// act(z).  The tanh form uses 1/2 (1 + tanh u) = sigmoid(2u), which keeps the
// relative accuracy of the left tail.  ReLU passes a NaN on.
template <int ACT>
__device__ __forceinline__ float activate(float z)
{
    if (ACT == CHPL_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (ACT == CHPL_ACT_GELU) {
        float E;
        return z * normal_cdf(z, E);
    }
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
        float E;
        const float cdf = normal_cdf(z, E);
        slope = cdf + z * (0.3989422804014327f * E);
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
// rows t0 .. t0 + NB - 1 (NB <= 32).  Every lane of the warp calls both halves.  Each store or
// load of a row is one coalesced access of the warp (64 bytes in 16 bits).
//
// What it reads (an addend, a pre-activation) is fetched in a call of its own,
// ahead of the accumulators, so that the loads run under the products or under
// the arithmetic of the previous rows: one round trip to memory per 16 rows,
// taken one after another, is longer than a tile's products.
template <int NB>
struct Fetched {
    uint32_t add[NB];  // raw bits: 16-bit, or FP32
    uint32_t z[NB];    // raw bits: 16-bit, or a code
    uint32_t scale;    // lane j: the scale of row j's group
};

template <typename T>
__device__ __forceinline__ float from_bits(uint32_t b)
{
    const unsigned short h = (unsigned short)b;
    return to_f32(reinterpret_cast<const T&>(h));
}

template <typename T, Kind KIND, int NB>
__device__ __forceinline__ void fetch(const Epilogue& e, int f, int t0, Fetched<NB>& x)
{
    const bool ok = f < e.m;
    const int nt = min(NB, e.n - t0);
    if (e.add) {
        if (KIND == kGradWeight && e.out_f32) {
            const uint32_t* a = static_cast<const uint32_t*>(e.add) + (int64_t)t0 * e.ldadd + f;
#pragma unroll
            for (int j = 0; j < NB; ++j) x.add[j] = ok && j < nt ? a[j * e.ldadd] : 0u;
        } else {
            const unsigned short* a = static_cast<const unsigned short*>(e.add) + (int64_t)t0 * e.ldadd + f;
#pragma unroll
            for (int j = 0; j < NB; ++j) x.add[j] = ok && j < nt ? a[j * e.ldadd] : 0u;
        }
    }
    if (KIND == kGradInput && e.act != CHPL_ACT_NONE) {
        if (e.z8.codes) {
            const uint8_t* c = reinterpret_cast<const uint8_t*>(e.z8.codes) + (int64_t)t0 * e.z8.ldc + f;
#pragma unroll
            for (int j = 0; j < NB; ++j) x.z[j] = ok && j < nt ? c[j * e.z8.ldc] : 0u;
            const int lane = lane_id(), g = f - lane;
            x.scale = g < e.m && lane < nt ? e.z8.scales[(int64_t)(t0 + lane) * e.z8.lds + g / kCkptGroup] : kCkptMinScale;
        } else {
            const unsigned short* z = static_cast<const unsigned short*>(e.z) + (int64_t)t0 * e.ldz + f;
#pragma unroll
            for (int j = 0; j < NB; ++j) x.z[j] = ok && j < nt ? z[j * e.ldz] : 0u;
        }
    }
}

template <typename T, int NB>
__device__ __forceinline__ void put_rows(void* out, int64_t ld, int f, int t0, int nt, const float (&v)[NB])
{
    T* o = static_cast<T*>(out) + (int64_t)t0 * ld + f;
#pragma unroll
    for (int j = 0; j < NB; ++j)
        if (j < nt) o[j * ld] = from_f32<T>(v[j]);
}

template <typename T, Kind KIND, int NB>
__device__ __forceinline__ void finish(const Epilogue& e, int f, int t0, float (&v)[NB], float bias, const Fetched<NB>& x)
{
    const bool ok = f < e.m;
    const int nt = ok ? min(NB, e.n - t0) : 0;  // rows this lane stores
    if (KIND == kGradWeight) {
        if (e.out_f32) {
            if (e.add) {
#pragma unroll
                for (int j = 0; j < NB; ++j) v[j] += __uint_as_float(x.add[j]);
            }
            put_rows<float, NB>(e.out, e.ldo, f, t0, nt, v);
            return;
        }
    } else if (KIND == kForward) {
#pragma unroll
        for (int j = 0; j < NB; ++j) v[j] += bias;
        if (e.z) put_rows<T, NB>(e.z, e.ldz, f, t0, nt, v);
        if (e.z8.codes) {
            const int lane = lane_id(), g = f - lane;
            int8_t* o = e.z8.codes + (int64_t)t0 * e.z8.ldc + f;
            uint32_t mine = 0;  // lane j: the scale of row j
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const uint32_t bits = ok ? __float_as_uint(v[j]) & 0x7fffffffu : 0u;
                const uint32_t s = ckpt_scale(__reduce_max_sync(0xffffffffu, bits));
                const uint32_t code = s == kCkptBadScale ? 0u : ckpt_code(v[j], ckpt_inv_step(s));
                mine = lane == j ? s : mine;
                if (j < nt) o[j * e.z8.ldc] = (int8_t)code;
            }
            if (g < e.m && lane < min(NB, e.n - t0))
                e.z8.scales[(int64_t)(t0 + lane) * e.z8.lds + g / kCkptGroup] = (uint8_t)mine;
        }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < NB; ++j) v[j] = activate<decltype(tag)::value>(v[j]);
        });
    } else if (e.act != CHPL_ACT_NONE) {
        float z[NB];
        if (e.z8.codes) {
            const float step = ckpt_step(x.scale);
#pragma unroll
            for (int j = 0; j < NB; ++j) z[j] = ckpt_value(x.z[j] ^ 0x80u, 0, __shfl_sync(0xffffffffu, step, j));
        } else {
#pragma unroll
            for (int j = 0; j < NB; ++j) z[j] = from_bits<T>(x.z[j]);
        }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                float slope;
                slope_and_value<decltype(tag)::value>(z[j], slope, z[j]);
                v[j] *= slope;
            }
        });
        if (e.xv) put_rows<T, NB>(e.xv, e.ldxv, f, t0, nt, z);
    }
    if (e.add) {
#pragma unroll
        for (int j = 0; j < NB; ++j) v[j] += from_bits<T>(x.add[j]);
    }
    put_rows<T, NB>(e.out, e.ldo, f, t0, nt, v);
}

template <typename T>
__device__ __forceinline__ float bias_of(const Epilogue& e, int f)
{
    return e.bias && f < e.m ? to_f32(static_cast<const T*>(e.bias)[f]) : 0.0f;
}

}  // namespace linear
}  // namespace chpl
