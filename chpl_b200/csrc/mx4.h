// Internal interface of the 4-bit module (mx4.cu, mx4_gemm.cu): where codes and
// scales lie, and their coding.
#pragma once

#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace mx4 {

constexpr int kGroup = 32;
constexpr uint32_t kMinScale = 5;    // of an all-zero group; keeps a step and its inverse normal FP32 numbers
constexpr uint32_t kBadScale = 255;  // the group held an infinity or a NaN
constexpr int kBlockRows = 128;      // of scales: kBlockRows x 4 groups are 512 consecutive bytes
constexpr int kBlockBytes = 512;
constexpr int kPiece = 256;          // columns that the products take at a time; scales come in whole pieces

// blocks of scales along a row: two to a piece
__host__ __device__ inline int64_t blocks_of(int64_t cols) { return (cols + kPiece - 1) / kPiece * 2; }
// bytes between rows of codes that lie close together: whole groups
inline int64_t code_bytes(int64_t cols) { return (cols + kGroup - 1) / kGroup * (kGroup / 2); }
inline int64_t scale_bytes(int64_t rows, int64_t cols) { return (rows + kBlockRows - 1) / kBlockRows * blocks_of(cols) * kBlockBytes; }

// where row t's groups 4 q .. 4 q + 3 have their scales
__device__ __forceinline__ int64_t scale_at(uint32_t t, int64_t q, int64_t blocks)
{
    return ((int64_t)(t / kBlockRows) * blocks + q) * kBlockBytes + (t % 32) * 16 + (t % kBlockRows) / 32 * 4;
}

// scale of a group from its largest magnitude's FP32 bits
__device__ __forceinline__ uint32_t scale_of(uint32_t max_bits)
{
    const uint32_t e = max_bits >> 23;
    return e == 255 ? kBadScale : max(e, kMinScale + 2) - 2;
}
// 2^(127 - s); 0 for a group whose codes are to be 0
__device__ __forceinline__ float inv_step(uint32_t s) { return s == kBadScale ? 0.0f : __uint_as_float((254u - s) << 23); }
// 2^(s - 127); NaN for a poisoned group.  s = 0, which no pack writes, is 2^-127.
__device__ __forceinline__ float step(uint32_t s)
{
    return s == kBadScale ? __uint_as_float(0x7fffffffu) : s == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}

// codes of v[0..7] times inv in nibbles 0..7: rounded to nearest, ties to the even
// code, magnitudes above 6 to 6
__device__ __forceinline__ uint32_t codes8(const float* v, float inv)
{
    uint32_t w;
    float q[8];
    const Two m = both(inv);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 p = apart(two(v[i], v[i + 1]) * m);
        q[i] = p.x;
        q[i + 1] = p.y;
    }
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return w;
}

// values of the codes in w, times the step
__device__ __forceinline__ void values8(uint32_t w, float st, float* v)
{
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(reinterpret_cast<const __half2&>(h[i]));
        v[2 * i] = f.x * st;
        v[2 * i + 1] = f.y * st;
    }
}

int check_mx4(const char* who, const char* what, const chpl_mx4& c, int64_t rows, int64_t cols);
int pack(cudaStream_t st, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4& c);

// Y = act(X W^T + b) + R, `type` of b, R and Y.  X comes in codes, or in 16 bits
// (x16, x.codes NULL), which the product then codes itself: up to kCodedRows rows.
constexpr int kCodedRows = 8;
int gemm(cudaStream_t st, int type, const chpl_mx4& w, const chpl_mx4& x, const void* x16, int64_t ldx, int64_t k, const linear::Epilogue& e);

int read_clear_status(int* st);

}  // namespace mx4
}  // namespace chpl
