// 8-bit activation checkpoints: pack and unpack (the C entry points
// chpl_ckpt8_pack / chpl_ckpt8_unpack).
//
// Bound: HBM.  A matrix of T x D elements of e bytes moves e T D + T D (1 +
// 1/32) bytes each way.
#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace linear {

constexpr int kPackThreads = 256;

// one warp per group of 32 features, a lane per feature
template <typename T>
__global__ void __launch_bounds__(kPackThreads) ckpt8_pack_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                                  int cols, int groups, chpl_ckpt8 c)
{
    const int lane = lane_id();
    const int64_t total = rows * groups, step = (int64_t)gridDim.x * (kPackThreads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kPackThreads / 32) + warp_id(); w < total; w += step) {
        const int64_t t = w / groups;
        const int g = (int)(w - t * groups), j = g * kCkptGroup + lane;
        const float v = j < cols ? to_f32(x[t * ldx + j]) : 0.0f;
        const uint32_t s = ckpt_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
        const int code = ckpt_code(v, ckpt_inv_step(s));
        if (j < cols) c.codes[t * c.ldc + j] = (int8_t)code;
        if (lane == 0) c.scales[t * c.lds + g] = (uint8_t)s;
    }
}

template <typename T>
__global__ void __launch_bounds__(kPackThreads) ckpt8_unpack_kernel(T* __restrict__ x, int64_t ldx, int64_t rows,
                                                                    int cols, int groups, chpl_ckpt8 c)
{
    const int lane = lane_id();
    const int64_t total = rows * groups, step = (int64_t)gridDim.x * (kPackThreads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kPackThreads / 32) + warp_id(); w < total; w += step) {
        const int64_t t = w / groups;
        const int g = (int)(w - t * groups), j = g * kCkptGroup + lane;
        if (j < cols) x[t * ldx + j] = from_f32<T>((float)c.codes[t * c.ldc + j] * ckpt_step(c.scales[t * c.lds + g]));
    }
}

static int check_matrix(const char* who, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                        const chpl_ckpt8* c)
{
    if (type != CHPL_TYPE_BF16 && type != CHPL_TYPE_F16 && type != CHPL_TYPE_F32) {
        set_error("%s: unknown type %d", who, type);
        return CHPL_ERR_INVALID;
    }
    CHPL_TRY(check_size(who, "rows", rows));
    CHPL_TRY(check_size(who, "cols", cols));
    if (!c) { set_error("%s: checkpoint is NULL", who); return CHPL_ERR_INVALID; }
    if (rows == 0 || cols == 0) return CHPL_OK;
    CHPL_TRY(check_operand(who, "x", x, ldx, cols, type == CHPL_TYPE_F32 ? 4 : 2));
    return check_ckpt(who, "checkpoint", *c, cols);
}

template <typename T>
static int pack(cudaStream_t st, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_ckpt8& c)
{
    const int groups = (int)((cols + kCkptGroup - 1) / kCkptGroup);
    ckpt8_pack_kernel<T><<<grid_for(rows * groups, kPackThreads / 32), kPackThreads, 0, st>>>(
        static_cast<const T*>(x), ldx, rows, (int)cols, groups, c);
    CHPL_CUDA(cudaGetLastError());
    return CHPL_OK;
}

template <typename T>
static int unpack(cudaStream_t st, int64_t rows, int64_t cols, void* x, int64_t ldx, const chpl_ckpt8& c)
{
    const int groups = (int)((cols + kCkptGroup - 1) / kCkptGroup);
    ckpt8_unpack_kernel<T><<<grid_for(rows * groups, kPackThreads / 32), kPackThreads, 0, st>>>(
        static_cast<T*>(x), ldx, rows, (int)cols, groups, c);
    CHPL_CUDA(cudaGetLastError());
    return CHPL_OK;
}

}  // namespace linear
}  // namespace chpl

extern "C" int chpl_ckpt8_pack(void* stream, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                               const chpl_ckpt8* c)
{
    using namespace chpl::linear;
    CHPL_TRY(check_matrix("ckpt8_pack", type, rows, cols, x, ldx, c));
    if (rows == 0 || cols == 0) return CHPL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == CHPL_TYPE_BF16) return pack<__nv_bfloat16>(st, rows, cols, x, ldx, *c);
    if (type == CHPL_TYPE_F16) return pack<__half>(st, rows, cols, x, ldx, *c);
    return pack<float>(st, rows, cols, x, ldx, *c);
}

extern "C" int chpl_ckpt8_unpack(void* stream, int type, int64_t rows, int64_t cols, const chpl_ckpt8* c, void* x,
                                 int64_t ldx)
{
    using namespace chpl::linear;
    CHPL_TRY(check_matrix("ckpt8_unpack", type, rows, cols, x, ldx, c));
    if (rows == 0 || cols == 0) return CHPL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == CHPL_TYPE_BF16) return unpack<__nv_bfloat16>(st, rows, cols, x, ldx, *c);
    if (type == CHPL_TYPE_F16) return unpack<__half>(st, rows, cols, x, ldx, *c);
    return unpack<float>(st, rows, cols, x, ldx, *c);
}
