// Activations, their slopes, and the epilogue of the linear-layer products.
#pragma once

#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace linear {

__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ Two ex2(Two a)
{
    const float2 x = apart(a);
    return two(ex2(x.x), ex2(x.y));
}
__device__ __forceinline__ Two rcp(Two a)
{
    const float2 x = apart(a);
    return two(rcp(x.x), rcp(x.y));
}

constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^-w), i.e. the logistic function of w / log2(e); 2^x and the
// reciprocal by the hardware's approximations (relative error below 2^-20
// where the result matters to 16 bits)
__device__ __forceinline__ Two logistic2(Two w) { return rcp(both(1.0f) + ex2(w * both(-1.0f))); }

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// Phi(z), the normal distribution function, and E = exp(-z^2 / 2) by the way:
// Abramowitz and Stegun 7.1.26 (Hastings), erfc(x) = t (a1 + ... + a5 t^4) E
// with t = 1 / (1 + p x), x = |z| / sqrt(2), absolute error below 1.5e-7.  One
// exponential and one reciprocal, and the slope's density is E again.  In the left
// tail the error is in E's proportion: relative 5e-5 at -3, 5e-4 at -4 (F16's unit),
// 1.6e-3 at -5 and 3.6e-3 at -6 (BF16's), where 1 + erf has cancelled in FP32.
__device__ __forceinline__ Two normal_cdf(Two z, Two& E)
{
    const float2 s = apart(z);
    E = ex2(z * (z * both(-0.5f * kLog2e)));
    const Two t = rcp(fma2(both(0.3275911f * 0.70710678f), two(fabsf(s.x), fabsf(s.y)), both(1.0f)));
    Two q = fma2(both(0.5f * 1.061405429f), t, both(0.5f * -1.453152027f));
    q = fma2(q, t, both(0.5f * 1.421413741f));
    q = fma2(q, t, both(0.5f * -0.284496736f));
    q = fma2(q, t, both(0.5f * 0.254829592f));
    const Two tail = (q * t) * E, head = fma2(tail, both(-1.0f), both(1.0f));
    const float2 a = apart(tail), b = apart(head);
    return two(s.x < 0.0f ? a.x : b.x, s.y < 0.0f ? a.y : b.y);
}

// act(z).  The tanh form uses 1/2 (1 + tanh u) = logistic(2u), which keeps the
// relative accuracy of the left tail.  ReLU passes a NaN on.
template <int ACT>
__device__ __forceinline__ void activate(float& a, float& b)
{
    if (ACT == CHPL_ACT_NONE) return;
    if (ACT == CHPL_ACT_RELU) {
        a = a < 0.0f ? 0.0f : a;
        b = b < 0.0f ? 0.0f : b;
        return;
    }
    const Two z = two(a, b);
    Two g, E;
    if (ACT == CHPL_ACT_GELU) g = normal_cdf(z, E);
    else if (ACT == CHPL_ACT_GELU_TANH)
        g = logistic2(z * fma2(z * z, both(2.0f * kLog2e * kGeluC * kGeluA), both(2.0f * kLog2e * kGeluC)));
    else g = logistic2(z * both(kLog2e));
    const float2 r = apart(z * g);
    a = r.x;
    b = r.y;
}

// act'(z) into s and act(z) into z, from the same transcendental.  Where the
// slope has settled, |z| above 20, its polynomial factors are held at 20 so that
// they cannot overflow against a zero.
__device__ __forceinline__ float hold20(float z) { return fminf(fmaxf(z, -20.0f), 20.0f); }

template <int ACT>
__device__ __forceinline__ void slope_and_value(float& za, float& zb, float& sa, float& sb)
{
    if (ACT == CHPL_ACT_NONE) {
        sa = sb = 1.0f;
        return;
    }
    if (ACT == CHPL_ACT_RELU) {
        sa = za > 0.0f ? 1.0f : 0.0f;
        sb = zb > 0.0f ? 1.0f : 0.0f;
        za = za < 0.0f ? 0.0f : za;
        zb = zb < 0.0f ? 0.0f : zb;
        return;
    }
    const Two z = two(za, zb);
    Two g, slope;
    if (ACT == CHPL_ACT_GELU) {
        Two E;
        g = normal_cdf(z, E);
        slope = fma2(z, E * both(0.3989422804014327f), g);
    } else {
        const Two zc = two(hold20(za), hold20(zb));
        if (ACT == CHPL_ACT_GELU_TANH) {
            g = logistic2(z * fma2(z * z, both(2.0f * kLog2e * kGeluC * kGeluA), both(2.0f * kLog2e * kGeluC)));
            const Two d = fma2(zc * zc, both(6.0f * kGeluC * kGeluA), both(2.0f * kGeluC));  // of 2u
            slope = fma2((zc * d) * g, fma2(g, both(-1.0f), both(1.0f)), g);
        } else {
            g = logistic2(z * both(kLog2e));
            slope = fma2(zc * g, fma2(g, both(-1.0f), both(1.0f)), g);
        }
    }
    float2 r = apart(slope);
    sa = r.x;
    sb = r.y;
    r = apart(z * g);
    za = r.x;
    zb = r.y;
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

// ----------------------------------------------------------------------------
// The epilogue of one warp: 32 features from f0 (a multiple of 32, so a warp
// holds whole checkpoint groups) by NCB blocks of 8 rows from t0.
//
// The accumulators come as tcgen05.ld's 16x256b fragments, laid out like an
// mma accumulator: element (h, cb, rr, p) of lane l is feature 16 h + 8 rr + l/4
// and row 8 cb + 2 (l % 4) + p.  A pair of rows packs into one register, so
// stmatrix / ldmatrix with .trans turn 8 x 8 blocks between fragments and rows
// of 8 consecutive features in shared memory, and global memory is read and
// written 16 bytes a lane: row l / 4 of a block, features 8 (l % 4) to + 7
// ("line" order).  Per 32 outputs that is about two instructions beyond the
// arithmetic; a store of 2 bytes per lane and row took over twenty and bounded
// every product with a short contraction.
//
// What the epilogue reads (an addend, a pre-activation) is fetched ahead of the
// accumulators: for a warp's first rows before it waits for them, for the others
// as soon as the rows before have taken theirs out of the registers.  READS is
// false where there is nothing to read.
// ----------------------------------------------------------------------------
// accumulators of 32 lanes (features) and NCB x 8 columns (rows t), as the
// fragments that the epilogue takes
template <int NCB>
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[8 * NCB])
{
    uint32_t r[8 * NCB];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NCB / 2; ++c) {
            uint32_t* q = r + (h * NCB + 2 * c) * 4;
            asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7])
                         : "r"(taddr + ((uint32_t)(16 * h) << 16) + 16 * c));
        }
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 8 * NCB; ++j) v[j] = __uint_as_float(r[j]);
}

// Arrival on the even CTA's barrier that this warp has read its accumulators
// (ordered by tcgen05.fence, not by the memory model: the default CTA-scope
// release does not wait for the stores under way, as a cluster-scope one would).
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

constexpr int kStageBytes = 2048;  // a warp's shared memory: 32 rows of 64 bytes

template <int NCB>
struct Fetched {
    uint4 add[NCB];          // line order, 16-bit
    float add32[8 * NCB];    // fragment order (FP32 gradients)
    uint4 z[NCB];            // line order: 16-bit, or codes in x and y
    uint32_t scale[NCB];     // of row l / 4 of each block
};

template <int NCB>
__device__ __forceinline__ constexpr int frag(int h, int cb, int rr, int p) { return (h * NCB + cb) * 4 + rr * 2 + p; }

// Lines of 16-bit rows t0 + 8 cb + l / 4, features f0 + 8 (l % 4) to + 7; zero
// where there are none.  Whole lines come without a branch among the loads.
template <int NCB>
__device__ __forceinline__ void lines16(const void* base, int64_t ld, int t0, int f0, int n, int m, bool vec, uint4 (&w)[NCB])
{
    const int lane = lane_id(), f = f0 + 8 * (lane & 3);
    const unsigned short* at = static_cast<const unsigned short*>(base) + (int64_t)(t0 + (lane >> 2)) * ld + f;
    if (vec && f0 + 32 <= m) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            w[cb] = make_uint4(0, 0, 0, 0);
            if (t0 + 8 * cb + (lane >> 2) < n) w[cb] = *reinterpret_cast<const uint4*>(at + 8 * cb * ld);
        }
        return;
    }
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        w[cb] = make_uint4(0, 0, 0, 0);
        uint32_t* u = &w[cb].x;
        if (t0 + 8 * cb + (lane >> 2) < n) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (f + i < m) u[i >> 1] |= (uint32_t)at[8 * cb * ld + i] << (16 * (i & 1));
        }
    }
}

// the same of a checkpoint: codes into x and y, the lines' scales
template <int NCB>
__device__ __forceinline__ void lines_ckpt(const chpl_ckpt8& c, int t0, int f0, int n, int m, bool vec, uint4 (&w)[NCB],
                                           uint32_t (&scale)[NCB])
{
    const int lane = lane_id(), f = f0 + 8 * (lane & 3);
    const int64_t t = t0 + (lane >> 2);
    const int8_t* at = c.codes + t * c.ldc + f;
    const uint8_t* sc = c.scales + t * c.lds + f0 / kCkptGroup;
    const bool whole = vec && f0 + 32 <= m;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        w[cb] = make_uint4(0, 0, 0, 0);
        scale[cb] = kCkptMinScale;
        if (t0 + 8 * cb + (lane >> 2) < n && f0 < m) {
            scale[cb] = sc[8 * cb * c.lds];
            if (whole) {
                const uint2 two = *reinterpret_cast<const uint2*>(at + 8 * cb * c.ldc);
                w[cb].x = two.x;
                w[cb].y = two.y;
            }
        }
    }
    if (whole) return;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        uint32_t* u = &w[cb].x;
        if (t0 + 8 * cb + (lane >> 2) < n) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (f + i < m) u[i >> 2] |= (uint32_t)(uint8_t)at[8 * cb * c.ldc + i] << (8 * (i & 3));
        }
    }
}

// where a warp goes after these rows; f0 < 0: nowhere
struct Next {
    int f0, t0;
};

template <typename T, Kind KIND, int NCB>
__device__ __forceinline__ void fetch(const Epilogue& e, int f0, int t0, Fetched<NCB>& x)
{
    const int lane = lane_id();
    if (e.add) {
        if (KIND == kGradWeight && e.out_f32) {
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int t = t0 + 8 * cb + 2 * (lane & 3) + p;
                    const float* a = static_cast<const float*>(e.add) + (int64_t)t * e.ldadd + f0 + (lane >> 2);
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        x.add32[frag<NCB>(g >> 1, cb, g & 1, p)] = t < e.n && f0 + (lane >> 2) + 8 * g < e.m ? a[8 * g] : 0.0f;
                }
        } else {
            lines16<NCB>(e.add, e.ldadd, t0, f0, e.n, e.m, e.vec_add, x.add);
        }
    }
    if (KIND == kGradInput && e.act != CHPL_ACT_NONE) {
        if (e.z8.codes) lines_ckpt<NCB>(e.z8, t0, f0, e.n, e.m, e.vec_codes, x.z, x.scale);
        else lines16<NCB>(e.z, e.ldz, t0, f0, e.n, e.m, e.vec_z, x.z);
    }
}

// byte offset of row t's features 8 c .. 8 c + 7 (16-bit) in a staged matrix of
// 64-byte rows: the 16-byte pieces of every other row are swapped about, so
// that eight rows' pieces fall into different banks
__device__ __forceinline__ uint32_t staged(int t, int c) { return (uint32_t)(t * 64 + ((c ^ ((t >> 1) & 3)) << 4)); }

// line order -> fragments of two rows each, through `at` (shared)
template <int NCB>
__device__ __forceinline__ void to_fragments(uint32_t at, const uint4 (&line)[NCB], uint32_t (&r)[4 * NCB])
{
    const int lane = lane_id();
    __syncwarp();  // the warp's reads of what was staged before are over
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + staged(8 * cb + (lane >> 2), lane & 3)),
                     "r"(line[cb].x), "r"(line[cb].y), "r"(line[cb].z), "r"(line[cb].w)
                     : "memory");
    __syncwarp();
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[4 * cb]), "=r"(r[4 * cb + 1]), "=r"(r[4 * cb + 2]), "=r"(r[4 * cb + 3])
                     : "r"(at + staged(8 * cb + (lane & 7), lane >> 3))
                     : "memory");
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
    return __half22float2(reinterpret_cast<const __half2&>(w));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
}

// v (fragments) as 16-bit rows of `out`, through `at` (shared)
template <typename T, int NCB>
__device__ __forceinline__ void put16(const Epilogue& e, void* out, int64_t ld, bool vec, int f0, int t0, uint32_t at,
                                      const float (&v)[8 * NCB])
{
    const int lane = lane_id();
    __syncwarp();
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        uint32_t w[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) w[g] = pack2<T>(v[frag<NCB>(g >> 1, cb, g & 1, 0)], v[frag<NCB>(g >> 1, cb, g & 1, 1)]);
        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                         at + staged(8 * cb + (lane & 7), lane >> 3)),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
    }
    __syncwarp();
    unsigned short* o = static_cast<unsigned short*>(out) + (int64_t)t0 * ld + f0;
    if (vec && f0 + 32 <= e.m) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            const int t = 8 * cb + (lane >> 2);
            uint4 w;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                         : "r"(at + staged(t, lane & 3))
                         : "memory");
            if (t0 + t < e.n) *reinterpret_cast<uint4*>(o + t * ld + 8 * (lane & 3)) = w;
        }
    } else {  // rows that 16-byte stores cannot start on, and the last features: a lane per feature
        const int rows = min(8 * NCB, e.n - t0);
        if (f0 + lane < e.m) {
#pragma unroll 4
            for (int t = 0; t < rows; ++t) {
                unsigned short w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at + staged(t, lane >> 3) + 2 * (lane & 7)) : "memory");
                o[t * ld + lane] = w;
            }
        }
    }
}

// ReLU's slope at a checkpoint hangs on whether a code is 0 or 1, and a quotient
// near to +-1/2 would let the tiling decide over it: the tensor cores' sums are off
// by several times what an FP32 sum is.  With ReLU those quotients are formed again
// from the operands (SETTLE): products exact in FP32, eight added there, the eights
// in FP64.  Of 4100 x 16384 x 4200's slopes 38 are off without it, 2 with it, and 4
// of an FP32 product.
//
// How near (tie_width): the tensor cores add 16 products at a time into an FP32
// accumulator by cutting, toward zero, half a unit in the last place or 0.36 2^-23
// of the partial sum in the mean.  The mean of the partial sums of random terms
// whose sum ends near zero has 0.29 s as its standard deviation, s = sqrt(sum x^2
// w^2): over a contraction of 16384, 1.3e-5 s (measured: 0.9 to 1.0e-5 s, in
// proportion to the contraction of one CTA, so 1/8 of it split in 8).  The largest
// of a group's 32 is below 1.2 s once in 4000 groups, so s is at most 107 steps
// else, and 2e-5 steps for each k-block of 64 are five of the measured deviations;
// short contractions, whose error hangs on single products, have 5e-5 on top.
// Random operands settle that way; sums whose terms cancel to far less than their
// group's others can be off by more, and then follow the tiling.
//
// A warp lists what is near in the half of its staging memory that NCB = 2 leaves
// free, kSettled of 8 rows of 32 features at most (so that data made of ties costs
// no more than a few times the product), and a CTA's warps settle all lists at its
// end; what no list takes up becomes 0, which is what a quotient at a tie rounds
// to.  8192 x 4096 x 16384: 855 us, 790 without settling; 4096 x 16384 x 4096: 489,
// 410; 777 x 1024 x 4096: 17.6, 14.3; one token x 4096 x 16384: 25.6, 23.8.  Settled
// by a warp where they turn up, they hold up the tiles behind: 957, 488, 17.0 and
// 25.1 us with a width a quarter of this.
constexpr int kSettled = 8;
constexpr int kListed = 126;
// Outputs of a product, for each warp that lists them, of which random operands leave
// eight near: 1/2 is met by 0.05 of the quotients for each unit of width (32 normal
// values under a common step); values beside outliers come nearer to eight times that.
inline double settle_share(float tie) { return 8.0 / (0.05 * tie); }

struct SettleList {
    int count, unused;
    int2 at[kListed];  // t, f
};
static_assert(sizeof(SettleList) <= kStageBytes / 2, "list");

inline float tie_width(int kblocks, int split) { return fminf(0.25f, 5e-5f + 2e-5f * (float)((kblocks + split - 1) / split)); }

// the products of c .. c + 7; rows lie on 16-byte boundaries, as TMA wants them
template <typename T>
__device__ __forceinline__ float eight(const T* __restrict__ a, const T* __restrict__ b, const uint4& u, const uint4& v, int c, int k)
{
    float part = 0.0f;
    if (c + 8 <= k) {
        const T *p = reinterpret_cast<const T*>(&u), *q = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int h = 0; h < 8; ++h) part = fmaf(to_f32(p[h]), to_f32(q[h]), part);
    } else {
        for (int h = c; h < k; ++h) part = fmaf(to_f32(a[h]), to_f32(b[h]), part);
    }
    return part;
}

// a warp's memory: its staging and, with SETTLE, its list behind that
__device__ __forceinline__ SettleList& list_of(uint8_t* areas, int warp)
{
    return *reinterpret_cast<SettleList*>(areas + warp * kStageBytes + kStageBytes / 2);
}

// Settles the lists of WARPS warps, after a barrier of these; sync() is that
// barrier.  All of them form two quotients at a time, so that one alone takes
// little; a thread finishes each.
template <typename T, int WARPS, typename Sync>
__device__ __forceinline__ void settle_all(const Epilogue& e, uint8_t* areas, int thread, Sync&& sync)
{
    constexpr int kBatch = 64, kStride = WARPS * 32 * 8;
    static_assert(kBatch * sizeof(double) <= kStageBytes / 2 && kBatch <= WARPS * 32, "partial sums");
    const int lane = lane_id();
    int w = 0, at = 0, left = 0;
    for (int v = 0; v < WARPS; ++v) left += list_of(areas, v).count;
    for (int batch; left > 0; left -= batch) {
        batch = min(kBatch, left);
        int2 mine = make_int2(0, 0);
        for (int i = 0; i < batch; i += 2) {
            const T *a[2], *b[2];
            double sum[2] = {0.0, 0.0};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (i + h < batch) {
                    while (at == list_of(areas, w).count) {
                        ++w;
                        at = 0;
                    }
                    const int2 p = list_of(areas, w).at[at++];
                    if (thread == i + h) mine = p;
                    a[h] = static_cast<const T*>(e.w) + (int64_t)p.y * e.ldw;
                    b[h] = static_cast<const T*>(e.x) + (int64_t)p.x * e.ldx;
                } else {
                    a[h] = a[0];
                    b[h] = b[0];
                }
            }
            for (int c = thread * 8; c < e.k; c += 2 * kStride) {
                uint4 u[2][2], v[2][2];
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (c + r * kStride + 8 <= e.k) {
                            u[h][r] = *reinterpret_cast<const uint4*>(a[h] + c + r * kStride);
                            v[h][r] = *reinterpret_cast<const uint4*>(b[h] + c + r * kStride);
                        }
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h) sum[h] += (double)eight<T>(a[h], b[h], u[h][r], v[h][r], c + r * kStride, e.k);
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) {
                sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], d);
                sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], d);
            }
            if (lane < 2) reinterpret_cast<double*>(areas + (thread >> 5) * kStageBytes)[i + lane] = lane ? sum[1] : sum[0];
        }
        sync();
        if (thread < batch) {
            const int t = mine.x, f = mine.y;
            const uint32_t s = *const_cast<volatile uint8_t*>(e.z8.scales + (int64_t)t * e.z8.lds + f / kCkptGroup);
            double z = e.bias ? (double)to_f32(static_cast<const T*>(e.bias)[f]) : 0.0;
#pragma unroll
            for (int v = 0; v < WARPS; ++v) z += reinterpret_cast<const double*>(areas + v * kStageBytes)[thread];
            e.z8.codes[(int64_t)t * e.z8.ldc + f] = (int8_t)max(-127, min(127, __double2int_rn(z * (double)ckpt_inv_step(s))));
        }
        sync();
    }
}

// how far the nearer of two quotients is from +-1/2
__device__ __forceinline__ float from_half(Two v, Two inv)
{
    const float2 q = apart(v * inv);
    return fminf(fabsf(fabsf(q.x) - 0.5f), fabsf(fabsf(q.y) - 0.5f));
}
__device__ __forceinline__ bool is_near(float v, float inv, float tie) { return fabsf(fabsf(v * inv) - 0.5f) < tie; }

// Puts the lanes' near quotients (bits of `near`; at(i, f, t): where the i-th is)
// on the warp's list, kSettled of them at most.  Every lane calls it.
template <typename At>
__device__ __forceinline__ void list_near(SettleList& list, uint32_t near, At&& at)
{
    const int from = list.count, to = min(kListed, from + kSettled);
    int count = from;
    for (uint32_t lanes = __ballot_sync(0xffffffffu, near != 0); lanes && count < to; lanes = __ballot_sync(0xffffffffu, near != 0)) {
        int f = 0, t = 0;
        if (near) at(__ffs(near) - 1, f, t);
        const int slot = count + __popc(lanes & ((1u << lane_id()) - 1u));
        if (near && slot < to) list.at[slot] = make_int2(t, f);
        near &= near - 1;
        count = min(to, count + __popc(lanes));
    }
    __syncwarp();
    if (lane_id() == 0) list.count = count;
    __syncwarp();
}

// Codes and scales of v, through `at` (shared, 32-byte rows); with SETTLE the
// quotients near +-1/2 go on the warp's list.
template <bool SETTLE, int NCB>
__device__ __forceinline__ void put_ckpt(const Epilogue& e, int f0, int t0, uint32_t at, const float (&v)[8 * NCB], SettleList* list)
{
    const int lane = lane_id();
    const bool whole = f0 + 32 <= e.m;
    // row r = 2 cb + p: its group is four features in this lane and those of the
    // lanes of the same l % 4.  Step by step over all rows, so that the
    // shuffles' latencies overlap.
    uint32_t scale[2 * NCB], worst = 0;
#pragma unroll
    for (int r = 0; r < 2 * NCB; ++r) {
        scale[r] = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t bits = __float_as_uint(v[frag<NCB>(g >> 1, r >> 1, g & 1, r & 1)]) & 0x7fffffffu;
            scale[r] = max(scale[r], whole || f0 + (lane >> 2) + 8 * g < e.m ? bits : 0u);
        }
    }
#pragma unroll
    for (int x = 4; x <= 16; x *= 2)
#pragma unroll
        for (int r = 0; r < 2 * NCB; ++r) scale[r] = max(scale[r], __shfl_xor_sync(0xffffffffu, scale[r], x));
#pragma unroll
    for (int r = 0; r < 2 * NCB; ++r) {
        scale[r] = ckpt_scale(scale[r]);
        worst = max(worst, scale[r]);
    }
    // two rows at a time
    constexpr int kZero = 0x4B400000;  // 3 * 2^22
    int code[8 * NCB];
    float nearest = 1.0f;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        const Two inv = two(ckpt_inv_step(scale[2 * cb]), ckpt_inv_step(scale[2 * cb + 1]));
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int i = frag<NCB>(g >> 1, cb, g & 1, 0);
            if (SETTLE) nearest = fminf(nearest, from_half(two(v[i], v[i + 1]), inv));
            const float2 q = apart(fma2(two(v[i], v[i + 1]), inv, both(12582912.0f)));
            code[8 * cb + g] = min(max(__float_as_int(q.x), kZero - 127), kZero + 127);
            code[8 * cb + 4 + g] = min(max(__float_as_int(q.y), kZero - 127), kZero + 127);
        }
    }
    const bool some = SETTLE && __any_sync(0xffffffffu, nearest < e.tie);
    if (SETTLE && nearest < e.tie) {
#pragma unroll
        for (int r = 0; r < 2 * NCB; ++r)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (is_near(v[frag<NCB>(g >> 1, r >> 1, g & 1, r & 1)], ckpt_inv_step(scale[r]), e.tie)) code[4 * r + g] = -128;  // no code
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 2 * NCB; ++r)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(at + (8 * (r >> 1) + 2 * (lane & 3) + (r & 1)) * 32 + (lane >> 2) + 8 * g),
                         "r"(code[4 * r + g])
                         : "memory");
    if (__any_sync(0xffffffffu, worst == kCkptBadScale)) {  // rows with an infinity or a NaN in the group: codes 0
#pragma unroll
        for (int i = 0; i < 2 * NCB; ++i)
            if (scale[i] == kCkptBadScale) {
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(at + (8 * (i >> 1) + 2 * (lane & 3) + (i & 1)) * 32 + (lane >> 2) + 8 * g),
                                 "r"(0u)
                                 : "memory");
            }
    }
    if (lane < 4) {
        uint8_t* o = e.z8.scales + (int64_t)(t0 + 2 * lane) * e.z8.lds + f0 / kCkptGroup;
#pragma unroll
        for (int i = 0; i < 2 * NCB; ++i) {
            const int t = 8 * (i >> 1) + (i & 1);
            if (t0 + 2 * lane + t < e.n) o[t * e.z8.lds] = (uint8_t)scale[i];
        }
    }
    __syncwarp();
    int8_t* o = e.z8.codes + (int64_t)t0 * e.z8.ldc + f0;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        const int t = 8 * cb + (lane >> 2), f = 8 * (lane & 3);
        uint2 w;
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(at + t * 32 + f) : "memory");
        if (SETTLE && some) {  // 0 for the time being, which is what a quotient at a tie rounds to
            const uint32_t lo = __vcmpeq4(w.x, 0x80808080u), hi = __vcmpeq4(w.y, 0x80808080u);
            w.x &= ~lo;
            w.y &= ~hi;
            uint32_t near = ((lo & 0x08040201u) * 0x01010101u >> 24 & 0xfu) | (hi & 0x08040201u) * 0x01010101u >> 24 << 4;
            near &= t0 + t < e.n && f0 + f < e.m ? (1u << min(8, e.m - f0 - f)) - 1u : 0u;
            list_near(*list, near, [&](int i, int& at_f, int& at_t) {
                at_f = f0 + f + i;
                at_t = t0 + t;
            });
        }
        if (t0 + t >= e.n) continue;
        if (e.vec_codes && whole) {
            *reinterpret_cast<uint2*>(o + t * e.z8.ldc + f) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (f0 + f + i < e.m) o[t * e.z8.ldc + f + i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
    }
}

// Every lane of the warp calls it.  bias[2 h + rr]; `stage`: kStageBytes of
// shared memory of the warp's own (shared-space address, 128-byte aligned).
// READS: x holds what these rows read, and what the rows `next` do on return.
// EXTRA: kForward lists the codes to settle, kGradInput adds the rows into sums
// (features f0 + 8 g + l / 4).
template <typename T, Kind KIND, bool READS, bool EXTRA, int NCB>
__device__ __forceinline__ void finish(const Epilogue& e, int f0, int t0, float (&v)[8 * NCB], const float (&bias)[4],
                                       Fetched<NCB>& x, Next next, uint32_t stage, float (&sums)[4], SettleList* list)
{
    static_assert(NCB * 8 * 64 <= kStageBytes / (KIND == kForward && EXTRA ? 2 : 1), "stage");
    const int lane = lane_id();
    const bool here = f0 < e.m && t0 < e.n;
    uint32_t add[4 * NCB], zf[4 * NCB];
    if (READS && here) {
        if (KIND == kGradWeight && e.out_f32) {
            if (e.add) {
#pragma unroll
                for (int i = 0; i < 8 * NCB; ++i) v[i] += x.add32[i];
            }
        } else if (e.add) {
            to_fragments<NCB>(stage, x.add, add);
        }
        if (KIND == kGradInput && e.act != CHPL_ACT_NONE) {
            if (e.z8.codes) {
                // a code times its step is exact in bf16, whatever T is
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb) {
                    const CkptIn::Raw r = {make_uint2(x.z[cb].x, x.z[cb].y), x.scale[cb]};
                    float z[8];
                    CkptIn{e.z8, e.vec_codes}.value(r, z);
                    x.z[cb] = make_uint4(pack2<__nv_bfloat16>(z[0], z[1]), pack2<__nv_bfloat16>(z[2], z[3]),
                                         pack2<__nv_bfloat16>(z[4], z[5]), pack2<__nv_bfloat16>(z[6], z[7]));
                }
            }
            to_fragments<NCB>(stage, x.z, zf);
        }
    }
    if (READS && next.f0 >= 0) fetch<T, KIND, NCB>(e, next.f0, next.t0, x);
    if (!here) return;
    if (KIND == kGradWeight && e.out_f32) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int t = t0 + 8 * cb + 2 * (lane & 3) + p;
                float* o = static_cast<float*>(e.out) + (int64_t)t * e.ldo + f0 + (lane >> 2);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (t < e.n && f0 + (lane >> 2) + 8 * g < e.m) o[8 * g] = v[frag<NCB>(g >> 1, cb, g & 1, p)];
            }
        return;
    }
    if (KIND == kForward) {
#pragma unroll
        for (int i = 0; i < 8 * NCB; ++i) v[i] += bias[(i / (4 * NCB)) * 2 + ((i >> 1) & 1)];
        if (e.z) put16<T, NCB>(e, e.z, e.ldz, e.vec_z, f0, t0, stage, v);
        if (e.z8.codes) put_ckpt<EXTRA, NCB>(e, f0, t0, stage, v, list);
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int i = 0; i < 8 * NCB; i += 2) activate<decltype(tag)::value>(v[i], v[i + 1]);
        });
    }
    if (KIND == kGradInput && READS && e.act != CHPL_ACT_NONE) {
        float z[8 * NCB];
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float2 two = e.z8.codes ? unpack2<__nv_bfloat16>(zf[4 * cb + g]) : unpack2<T>(zf[4 * cb + g]);
                z[frag<NCB>(g >> 1, cb, g & 1, 0)] = two.x;
                z[frag<NCB>(g >> 1, cb, g & 1, 1)] = two.y;
            }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int i = 0; i < 8 * NCB; i += 2) {
                float sa, sb;
                slope_and_value<decltype(tag)::value>(z[i], z[i + 1], sa, sb);
                v[i] *= sa;
                v[i + 1] *= sb;
            }
        });
        if (e.xv) put16<T, NCB>(e, e.xv, e.ldxv, true, f0, t0, stage, z);
    }
    if (READS && e.add) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float2 two = unpack2<T>(add[4 * cb + g]);
                v[frag<NCB>(g >> 1, cb, g & 1, 0)] += two.x;
                v[frag<NCB>(g >> 1, cb, g & 1, 1)] += two.y;
            }
    }
    if (KIND == kGradInput && EXTRA) {  // rows past the end are 0 x W: NaN where W is infinite
        const bool whole = t0 + 8 * NCB <= e.n;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 2 * NCB; ++i)
                sums[g] += whole || t0 + 8 * (i >> 1) + 2 * (lane & 3) + (i & 1) < e.n ? v[frag<NCB>(g >> 1, i >> 1, g & 1, i & 1)] : 0.0f;
    }
    put16<T, NCB>(e, e.out, e.ldo, e.vec_out, f0, t0, stage, v);
}

// ----------------------------------------------------------------------------
// The same epilogue where a warp holds one row, a lane four consecutive
// features (the joined sums of a split): memory is read and written 8 bytes a
// lane, a checkpoint group is eight lanes.
// ----------------------------------------------------------------------------
struct RowFetched {
    uint2 add;        // four 16-bit elements
    float4 add32;     // FP32 gradients
    uint2 z;          // four 16-bit elements, or codes in x
    uint32_t scale;
};

__device__ __forceinline__ uint2 row16(const void* base, int64_t ld, int t, int f, int n, int m, bool vec)
{
    uint2 w = make_uint2(0, 0);
    if (t >= n || f >= m) return w;
    const unsigned short* at = static_cast<const unsigned short*>(base) + (int64_t)t * ld + f;
    if (vec && f + 4 <= m) return *reinterpret_cast<const uint2*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (f + i < m) (i < 2 ? w.x : w.y) |= (uint32_t)at[i] << (16 * (i & 1));
    return w;
}

template <Kind KIND>
__device__ __forceinline__ void fetch_row(const Epilogue& e, int f, int t, RowFetched& x)
{
    if (e.add) {
        if (KIND == kGradWeight && e.out_f32) {
            float* v = &x.add32.x;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = t < e.n && f + i < e.m ? static_cast<const float*>(e.add)[(int64_t)t * e.ldadd + f + i] : 0.0f;
        } else {
            x.add = row16(e.add, e.ldadd, t, f, e.n, e.m, e.vec_add);
        }
    }
    if (KIND == kGradInput && e.act != CHPL_ACT_NONE) {
        if (!e.z8.codes) {
            x.z = row16(e.z, e.ldz, t, f, e.n, e.m, e.vec_z);
        } else {
            x.z = make_uint2(0, 0);
            x.scale = kCkptMinScale;
            if (t < e.n && f < e.m) {
                const int8_t* c = e.z8.codes + (int64_t)t * e.z8.ldc + f;
                x.scale = e.z8.scales[(int64_t)t * e.z8.lds + f / kCkptGroup];
                if (e.vec_codes && f + 4 <= e.m) {
                    x.z.x = *reinterpret_cast<const uint32_t*>(c);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (f + i < e.m) x.z.x |= (uint32_t)(uint8_t)c[i] << (8 * i);
                }
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void put_row16(void* out, int64_t ld, bool vec, int f, int t, int m, const float (&v)[4])
{
    T* o = static_cast<T*>(out) + (int64_t)t * ld + f;
    if (vec && f + 4 <= m) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f + i < m) o[i] = from_f32<T>(v[i]);
    }
}

// Every lane of the warp calls it; t < e.n; bias of the four features.
template <typename T, Kind KIND, bool READS, bool EXTRA>
__device__ __forceinline__ void finish_row(const Epilogue& e, int f, int t, float (&v)[4], const float (&bias)[4], const RowFetched& x,
                                           float (&sums)[4], SettleList* list)
{
    if (KIND == kGradWeight && e.out_f32) {
        float* o = static_cast<float*>(e.out) + (int64_t)t * e.ldo + f;
        if (READS && e.add) {
            v[0] += x.add32.x;
            v[1] += x.add32.y;
            v[2] += x.add32.z;
            v[3] += x.add32.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f + i < e.m) o[i] = v[i];
        return;
    }
    if (KIND == kForward) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += bias[i];
        if (e.z) put_row16<T>(e.z, e.ldz, e.vec_z, f, t, e.m, v);
        if (e.z8.codes) {
            uint32_t s = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) s = max(s, f + i < e.m ? __float_as_uint(v[i]) & 0x7fffffffu : 0u);
#pragma unroll
            for (int d = 1; d <= 4; d *= 2) s = max(s, __shfl_xor_sync(0xffffffffu, s, d));
            s = ckpt_scale(s);
            const float inv = ckpt_inv_step(s);
            uint32_t w = ckpt_codes4(v, inv);
            if (EXTRA) {
                const float nearest = fminf(from_half(two(v[0], v[1]), both(inv)), from_half(two(v[2], v[3]), both(inv)));
                if (__any_sync(0xffffffffu, nearest < e.tie)) {
                    uint32_t near = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (f + i < e.m && is_near(v[i], inv, e.tie)) {
                            near |= 1u << i;
                            w &= ~(0xffu << (8 * i));
                        }
                    list_near(*list, near, [&](int i, int& at_f, int& at_t) {
                        at_f = f + i;
                        at_t = t;
                    });
                }
            }
            if (s == kCkptBadScale) w = 0;
            int8_t* c = e.z8.codes + (int64_t)t * e.z8.ldc + f;
            if (e.vec_codes && f + 4 <= e.m) {
                *reinterpret_cast<uint32_t*>(c) = w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (f + i < e.m) c[i] = (int8_t)(w >> (8 * i));
            }
            if (f % kCkptGroup == 0 && f < e.m) e.z8.scales[(int64_t)t * e.z8.lds + f / kCkptGroup] = (uint8_t)s;
        }
        with_act(e.act, [&](auto tag) {
            activate<decltype(tag)::value>(v[0], v[1]);
            activate<decltype(tag)::value>(v[2], v[3]);
        });
    }
    if (KIND == kGradInput && READS && e.act != CHPL_ACT_NONE) {
        float z[4];
        if (e.z8.codes) {
            ckpt_values(x.z.x, ckpt_step(x.scale), z);
        } else {
            const float2 a = unpack2<T>(x.z.x), b = unpack2<T>(x.z.y);
            z[0] = a.x;
            z[1] = a.y;
            z[2] = b.x;
            z[3] = b.y;
        }
        with_act(e.act, [&](auto tag) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                float sa, sb;
                slope_and_value<decltype(tag)::value>(z[i], z[i + 1], sa, sb);
                v[i] *= sa;
                v[i + 1] *= sb;
            }
        });
        if (e.xv) put_row16<T>(e.xv, e.ldxv, true, f, t, e.m, z);
    }
    if (READS && e.add) {
        const float2 a = unpack2<T>(x.add.x), b = unpack2<T>(x.add.y);
        v[0] += a.x;
        v[1] += a.y;
        v[2] += b.x;
        v[3] += b.y;
    }
    if (KIND == kGradInput && EXTRA) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] += v[i];
    }
    put_row16<T>(e.out, e.ldo, e.vec_out, f, t, e.m, v);
}

// sums of a warp's rows into part `part` of e.sums
__device__ __forceinline__ void put_sums(const Epilogue& e, int part, int f0, float (&sums)[4])
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
        const int f = f0 + 8 * g + (lane_id() >> 2);
        if ((lane_id() & 3) == 0 && f < e.m) e.sums[(int64_t)part * e.m + f] = sums[g];
        sums[g] = 0.0f;
    }
}

// whether an epilogue does EXTRA, and whether it reads anything but the
// accumulators and the bias
inline bool extra(Kind kind, const Epilogue& e)
{
    if (kind == kGradInput) return e.sums != nullptr;
    return kind == kForward && e.z8.codes && e.act == CHPL_ACT_RELU;
}
inline bool reads(Kind kind, const Epilogue& e) { return e.add || (kind == kGradInput && e.act != CHPL_ACT_NONE); }

// the biases of a lane's four features of f0 .. f0 + 31
template <typename T>
__device__ __forceinline__ void bias_of(const Epilogue& e, int f0, float (&b)[4])
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int f = f0 + 8 * g + (lane_id() >> 2);
        b[g] = e.bias && f < e.m ? to_f32(static_cast<const T*>(e.bias)[f]) : 0.0f;
    }
}

}  // namespace linear
}  // namespace chpl
