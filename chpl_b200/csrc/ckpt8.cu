// 8-bit activation checkpoints: pack and unpack (the C entry points
// chpl_ckpt8_pack / chpl_ckpt8_unpack).
//
// Bound: HBM.  A matrix of T x D elements of e bytes moves e T D + T D (1 +
// 1/32) bytes each way.
#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace linear {

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
    return run_rows(st, RowsJob<RowsIn<T>, CkptOut, Keep>(rows_in<T>(x, ldx), ckpt_out(c), Keep(), rows, cols));
}

template <typename T>
static int unpack(cudaStream_t st, int64_t rows, int64_t cols, void* x, int64_t ldx, const chpl_ckpt8& c)
{
    return run_rows(st, RowsJob<CkptIn, RowsOut<T>, Keep>(ckpt_in(c), rows_out<T>(x, ldx), Keep(), rows, cols));
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
