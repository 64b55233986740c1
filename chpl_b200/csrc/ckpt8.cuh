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

#include <cstring>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace chpl {

// Kernels of these modules are launched with programmatic stream serialization:
// a kernel's blocks may start, and set themselves up, while the last ones of the
// kernel before it finish.  start_of_inputs() stands before a kernel's first
// access to global memory and waits until that kernel has completed; every
// thread calls it.  It first lets the next kernel in the same way.
__device__ __forceinline__ void start_of_inputs()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... P, typename... A>
int launch_kernel(void (*kernel)(P...), int64_t grid, int threads, int smem, int cluster, cudaStream_t st, A&&... args)
{
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    std::memset(&cfg, 0, sizeof(cfg));
    std::memset(attr, 0, sizeof(attr));
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CHPL_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
    return CHPL_OK;
}

// Two FP32 values in one register pair: Blackwell's packed add, multiply and
// fused multiply-add take one issue slot for both.  Each half rounds as the
// scalar instruction does.
struct Two {
    uint64_t v;
};

__device__ __forceinline__ Two two(float lo, float hi)
{
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ float2 apart(Two a)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b)
{
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b)
{
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

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

// Codes: x * inv is exact (a power of two; what could underflow is far below
// half a code), and adding 3 * 2^22 in the same instruction rounds it half to
// even into the sum's low mantissa bits, a 16-bit integer there (no conversion
// instruction, which runs at an eighth of an addition's rate); a clamp keeps it
// within +-127.  A poisoned group's codes are not numbers' and have to be
// replaced by 0.

// codes of v[0..3] in bytes 0..3
__device__ __forceinline__ uint32_t ckpt_codes4(const float* v, float inv)
{
    uint32_t h[2];  // as pairs of 16-bit integers
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 q = apart(fma2(two(v[2 * i], v[2 * i + 1]), both(inv), both(12582912.0f)));
        h[i] = __vmins2(__vmaxs2(__byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x5410), 0xff81ff81u), 0x007f007fu);
    }
    return __byte_perm(h[0], h[1], 0x6420);
}

// Values of the codes in bytes 0..3 of w: each, biased by 128, as the low byte of
// 2^23's mantissa, less 2^23 + 128, times the step; exact.
__device__ __forceinline__ void ckpt_values(uint32_t w, float step, float* v)
{
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const Two f = two(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | i)),
                          __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | (i + 1))));
        const float2 r = apart((f + both(-8388736.0f)) * both(step));
        v[i] = r.x;
        v[i + 1] = r.y;
    }
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

// ----------------------------------------------------------------------------
// Eight consecutive elements of a row, as one lane of rows_kernel holds them:
// raw() issues the loads, value() converts.  `vec`: base and row distance allow
// one 16-byte (8-byte for codes) access per lane; other rows, and a row's end,
// are read and written element by element.
// ----------------------------------------------------------------------------
template <typename T>
struct RowsIn {
    const T* p;
    int64_t ld;
    bool vec;
    struct Raw {
        uint4 w[sizeof(T) / 2];
    };
    __device__ __forceinline__ Raw raw(int64_t t, int j, int cols) const
    {
        Raw r;
        const T* at = p + t * ld + j;
        if (vec && j + 8 <= cols) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
        } else {
            T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = j + i < cols ? at[i] : from_f32<T>(0.0f);
        }
        return r;
    }
    __device__ __forceinline__ void value(const Raw& r, float (&v)[8]) const
    {
        const T* e = reinterpret_cast<const T*>(r.w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    }
    // the largest magnitude's FP32 bits; 16-bit patterns (sign cleared) order as
    // their values do, NaN on top, so two at a time compare as integers
    __device__ __forceinline__ uint32_t top(const Raw& r) const
    {
        if (sizeof(T) == 4) {
            uint32_t t = 0;
            const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
            for (int i = 0; i < 8; ++i) t = max(t, w[i] & 0x7fffffffu);
            return t;
        }
        const uint32_t t = __vmaxu2(__vmaxu2(r.w[0].x & 0x7fff7fffu, r.w[0].y & 0x7fff7fffu),
                                    __vmaxu2(r.w[0].z & 0x7fff7fffu, r.w[0].w & 0x7fff7fffu));
        const unsigned short h = (unsigned short)max(t & 0xffffu, t >> 16);
        return __float_as_uint(to_f32(reinterpret_cast<const T&>(h)));
    }
};

struct CkptIn {
    chpl_ckpt8 c;
    bool vec;
    struct Raw {
        uint2 w;
        uint32_t s;
    };
    __device__ __forceinline__ Raw raw(int64_t t, int j, int cols) const
    {
        Raw r = {make_uint2(0, 0), kCkptMinScale};
        if (j >= cols) return r;
        const int8_t* at = c.codes + t * c.ldc + j;
        r.s = c.scales[t * c.lds + j / kCkptGroup];
        if (vec && j + 8 <= cols) {
            r.w = __ldg(reinterpret_cast<const uint2*>(at));
        } else {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= (j + i < cols ? (uint32_t)(uint8_t)at[i] : 0u) << (8 * (i & 3));
            r.w = make_uint2(w[0], w[1]);
        }
        return r;
    }
    __device__ __forceinline__ void value(const Raw& r, float (&v)[8]) const
    {
        const float step = ckpt_step(r.s);
        ckpt_values(r.w.x, step, v);
        ckpt_values(r.w.y, step, v + 4);
    }
};

template <typename T>
struct RowsOut {
    T* p;
    int64_t ld;
    bool vec;
    __device__ __forceinline__ void put(int64_t t, int j, int cols, const float (&v)[8]) const
    {
        T* at = p + t * ld + j;
        uint4 w[sizeof(T) / 2];
        T* e = reinterpret_cast<T*>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
        if (vec && j + 8 <= cols) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(at)[i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < cols) at[i] = e[i];
        }
    }
    // the same for a whole warp, whose lanes hold 256 consecutive elements: rows
    // that pieces cannot start on are turned about in shared memory (`turn`, 256
    // elements of the warp's own), so that a store covers 32 elements in a row
    __device__ __forceinline__ void put_warp(int64_t t, int j, int cols, const float (&v)[8], void* turn) const
    {
        if (vec) return put(t, j, cols, v);
        T* buf = static_cast<T*>(turn);
        const int lane = lane_id(), j0 = j - lane * 8;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) buf[lane * 8 + i] = from_f32<T>(v[i]);
        __syncwarp();
        T* row = p + t * ld + j0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j0 + i * 32 + lane < cols) row[i * 32 + lane] = buf[i * 32 + lane];
    }
};

struct CkptOut {
    chpl_ckpt8 c;
    bool vec;
    // v and the largest magnitude's bits among them; every lane of a group's four
    // calls it; elements past the row's end are 0
    __device__ __forceinline__ void put(int64_t t, int j, int cols, const float (&v)[8], uint32_t top) const
    {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t s = ckpt_scale(top);
        const float inv = ckpt_inv_step(s);
        uint2 w = make_uint2(ckpt_codes4(v, inv), ckpt_codes4(v + 4, inv));
        if (s == kCkptBadScale) w = make_uint2(0, 0);
        if (j >= cols) return;
        int8_t* at = c.codes + t * c.ldc + j;
        if (vec && j + 8 <= cols) {
            *reinterpret_cast<uint2*>(at) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < cols) at[i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
        if (j % kCkptGroup == 0) c.scales[t * c.lds + j / kCkptGroup] = (uint8_t)s;
    }
};

inline bool aligned(const void* p, int64_t ld_bytes, int to)
{
    return reinterpret_cast<uintptr_t>(p) % to == 0 && ld_bytes % to == 0;
}
template <typename T>
RowsIn<T> rows_in(const void* p, int64_t ld) { return {static_cast<const T*>(p), ld, aligned(p, ld * (int64_t)sizeof(T), 16)}; }
template <typename T>
RowsOut<T> rows_out(void* p, int64_t ld) { return {static_cast<T*>(p), ld, aligned(p, ld * (int64_t)sizeof(T), 16)}; }
inline CkptIn ckpt_in(const chpl_ckpt8& c) { return {c, aligned(c.codes, c.ldc, 8)}; }
inline CkptOut ckpt_out(const chpl_ckpt8& c) { return {c, aligned(c.codes, c.ldc, 8)}; }

// out = f(in), row by row (a checkpoint takes in as it is): a warp takes UNITS x
// 256 columns of a row at a time, a lane 8 consecutive ones of each, every load
// before any arithmetic.
constexpr int kRowsThreads = 256;

struct Keep {
    __device__ __forceinline__ void operator()(float (&)[8]) const {}
};

template <typename In_, typename Out_, typename F_>
struct RowsJob {
    using In = In_;
    using Out = Out_;
    In in;
    Out out;
    F_ f;
    int64_t items;   // pieces of rows
    uint32_t segs;   // pieces of a row
    int cols;
    unsigned blocks;
    bool wide;       // pieces of UNITS units, else of one

    // units of a long row's piece: 64 bytes a lane under way
    static constexpr int kUnits = std::is_same<In, CkptIn>::value ? 8 : 4;

    RowsJob(const In& i, const Out& o, const F_& fn, int64_t rows, int64_t ncols) : in(i), out(o), f(fn), cols((int)ncols)
    {
        constexpr int64_t kBlocks = 148 * 8, kWarps = kRowsThreads / 32;  // eight resident blocks per SM, then a grid stride
        // long rows in pieces of several units, as long as that leaves every warp a piece
        const int64_t segs_wide = (ncols + kUnits * 256 - 1) / (kUnits * 256);
        wide = ncols > 256 && rows * segs_wide >= kBlocks * kWarps;
        segs = (uint32_t)(wide ? segs_wide : (ncols + 255) / 256);
        items = rows * segs;
        const int64_t want = (items + kWarps - 1) / kWarps;
        blocks = (unsigned)(want < kBlocks ? want : kBlocks);
    }

    template <int UNITS>
    __device__ __forceinline__ void run(unsigned block) const
    {
        __shared__ uint4 turns[kRowsThreads / 32][64];  // 256 elements of up to 4 bytes for each warp
        const int lane = lane_id();
        uint4* turn = turns[warp_id()];
        const int64_t step = (int64_t)blocks * (kRowsThreads / 32);
        for (int64_t i = (int64_t)block * (kRowsThreads / 32) + warp_id(); i < items; i += step) {
            const int64_t t = items < 0xffffffffll ? (int64_t)((uint32_t)i / segs) : i / segs;
            const int j0 = (int)(i - t * segs) * (UNITS * 256) + lane * 8;
            typename In::Raw raw[UNITS];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) raw[u] = in.raw(t, j0 + u * 256, cols);
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                float v[8];
                in.value(raw[u], v);
                f(v);
                if constexpr (std::is_same<Out, CkptOut>::value) out.put(t, j0 + u * 256, cols, v, in.top(raw[u]));
                else out.put_warp(t, j0 + u * 256, cols, v, turn);
            }
        }
    }
};

template <int UNITS, typename Job>
__global__ void __launch_bounds__(kRowsThreads) rows_kernel(const Job job)
{
    start_of_inputs();
    job.template run<UNITS>(blockIdx.x);
}

// two jobs side by side
template <typename A, typename B>
__global__ void __launch_bounds__(kRowsThreads) rows_pair_kernel(const A a, const B b)
{
    start_of_inputs();
    if (blockIdx.x < a.blocks) a.template run<1>(blockIdx.x);
    else b.template run<1>(blockIdx.x - a.blocks);
}

template <typename Job>
int run_rows(cudaStream_t st, const Job& job)
{
    return launch_kernel(job.wide ? rows_kernel<Job::kUnits, Job> : rows_kernel<1, Job>, job.blocks, kRowsThreads, 0, 1, st, job);
}

// small ones in one launch
template <typename A, typename B>
int run_rows(cudaStream_t st, const A& a, const B& b)
{
    if (!a.wide && !b.wide)
        return launch_kernel(rows_pair_kernel<A, B>, (int64_t)a.blocks + b.blocks, kRowsThreads, 0, 1, st, a, b);
    CHPL_TRY(run_rows(st, a));
    return run_rows(st, b);
}

}  // namespace chpl
