// Microscaled 4-bit floating point (OCP MXFP4): pack and unpack, and the C entry
// points chpl_mx4_pack, chpl_mx4_unpack and chpl_mx4_linear.
//
// Bound: HBM.  A matrix of T x D elements of e bytes moves e T D + T D (1 / 2 +
// 1 / 32) bytes each way.
#include "mx4.h"

namespace chpl {
namespace mx4 {

using linear::check_operand;
using linear::check_size;

int check_mx4(const char* who, const char* what, const chpl_mx4& c, int64_t rows, int64_t cols)
{
    CHPL_TRY(check_operand(who, what, c.codes, c.ldc, code_bytes(cols), 1));
    if (!aligned(c.codes, rows > 1 ? c.ldc : 0, 16)) { set_error("%s: rows of %s do not start on 16 bytes", who, what); return CHPL_ERR_INVALID; }
    if (!c.scales || reinterpret_cast<uintptr_t>(c.scales) % 16) { set_error("%s: scales of %s are NULL or not 16-byte aligned", who, what); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

static int check_matrix(const char* who, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4* c)
{
    if (type != CHPL_TYPE_BF16 && type != CHPL_TYPE_F16 && type != CHPL_TYPE_F32) { set_error("%s: unknown type %d", who, type); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_size(who, "rows", rows));
    CHPL_TRY(check_size(who, "cols", cols));
    if (!c) { set_error("%s: codes are NULL", who); return CHPL_ERR_INVALID; }
    if (rows == 0 || cols == 0) return CHPL_OK;
    CHPL_TRY(check_operand(who, "x", x, ldx, cols, type == CHPL_TYPE_F32 ? 4 : 2));
    return check_mx4(who, "the codes", *c, rows, cols);
}

template <typename T>
static int pack(cudaStream_t st, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4& c)
{
    return run_rows(st, RowsJob<RowsIn<T>, Out, Keep>(rows_in<T>(x, ldx), out(c, cols), Keep(), rows, cols));
}

template <typename T>
static int unpack(cudaStream_t st, int64_t rows, int64_t cols, void* x, int64_t ldx, const chpl_mx4& c)
{
    return run_rows(st, RowsJob<In, RowsOut<T>, Keep>(in(c, cols), rows_out<T>(x, ldx), Keep(), rows, cols));
}

int pack(cudaStream_t st, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4& c)
{
    if (type == CHPL_TYPE_BF16) return pack<__nv_bfloat16>(st, rows, cols, x, ldx, c);
    if (type == CHPL_TYPE_F16) return pack<__half>(st, rows, cols, x, ldx, c);
    return pack<float>(st, rows, cols, x, ldx, c);
}

// the workspace: codes and scales of X, where it comes in 16 bits
struct Plan {
    size_t scales = 0, bytes = 0;
};

static Plan plan(const chpl_mx4_fwd& a)
{
    Plan p;
    if (a.x4.codes || a.tokens == 0 || a.n == 0 || a.k == 0) return p;
    p.scales = round_up((size_t)(a.tokens * code_bytes(a.k)), 256);
    p.bytes = p.scales + round_up((size_t)scale_bytes(a.tokens, a.k), 256);
    return p;
}

static int check(const char* who, const chpl_mx4_fwd* a, bool pointers)
{
    if (!a) { set_error("%s: arguments are NULL", who); return CHPL_ERR_INVALID; }
    if (a->type != CHPL_TYPE_BF16 && a->type != CHPL_TYPE_F16) { set_error("%s: type %d is not BF16 or F16", who, a->type); return CHPL_ERR_INVALID; }
    if (a->act < CHPL_ACT_NONE || a->act > CHPL_ACT_SILU) { set_error("%s: unknown activation %d", who, a->act); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_size(who, "tokens", a->tokens));
    CHPL_TRY(check_size(who, "n", a->n));
    CHPL_TRY(check_size(who, "k", a->k));
    if (!pointers || a->tokens == 0 || a->n == 0) return CHPL_OK;
    if (a->k > 0) {
        if (a->x4.codes) CHPL_TRY(check_mx4(who, "x", a->x4, a->tokens, a->k));
        else CHPL_TRY(check_operand(who, "x", a->x, a->ldx, a->k, 2));
        CHPL_TRY(check_mx4(who, "w", a->w4, a->n, a->k));
    }
    CHPL_TRY(check_operand(who, "y", a->y, a->ldy, a->n, 2));
    if (a->bias) CHPL_TRY(check_operand(who, "bias", a->bias, a->n, a->n, 2));
    if (a->residual) CHPL_TRY(check_operand(who, "residual", a->residual, a->ldr, a->n, 2));
    if (a->y == a->residual && a->ldy != a->ldr) { set_error("%s: y is residual with another row distance", who); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

}  // namespace mx4
}  // namespace chpl

extern "C" int chpl_mx4_scale_bytes(int64_t rows, int64_t cols, int64_t* bytes)
{
    using namespace chpl::mx4;
    CHPL_TRY(check_size("mx4_scale_bytes", "rows", rows));
    CHPL_TRY(check_size("mx4_scale_bytes", "cols", cols));
    if (!bytes) { chpl::set_error("mx4_scale_bytes: bytes is NULL"); return CHPL_ERR_INVALID; }
    *bytes = scale_bytes(rows, cols);
    return CHPL_OK;
}

extern "C" int chpl_mx4_pack(void* stream, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4* c)
{
    using namespace chpl::mx4;
    CHPL_TRY(check_matrix("mx4_pack", type, rows, cols, x, ldx, c));
    if (rows == 0 || cols == 0) return CHPL_OK;
    return pack(static_cast<cudaStream_t>(stream), type, rows, cols, x, ldx, *c);
}

extern "C" int chpl_mx4_unpack(void* stream, int type, int64_t rows, int64_t cols, const chpl_mx4* c, void* x, int64_t ldx)
{
    using namespace chpl::mx4;
    CHPL_TRY(check_matrix("mx4_unpack", type, rows, cols, x, ldx, c));
    if (rows == 0 || cols == 0) return CHPL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == CHPL_TYPE_BF16) return unpack<__nv_bfloat16>(st, rows, cols, x, ldx, *c);
    if (type == CHPL_TYPE_F16) return unpack<__half>(st, rows, cols, x, ldx, *c);
    return unpack<float>(st, rows, cols, x, ldx, *c);
}

extern "C" int chpl_mx4_linear_worksize(const chpl_mx4_fwd* a, size_t* work_bytes)
{
    using namespace chpl::mx4;
    CHPL_TRY(check("mx4_linear_worksize", a, false));
    if (!work_bytes) { chpl::set_error("mx4_linear_worksize: work_bytes is NULL"); return CHPL_ERR_INVALID; }
    *work_bytes = plan(*a).bytes;
    return CHPL_OK;
}

extern "C" int chpl_mx4_linear(void* stream, const chpl_mx4_fwd* a, void* work, size_t work_bytes)
{
    using namespace chpl::mx4;
    CHPL_TRY(check("mx4_linear", a, true));
    if (a->tokens == 0 || a->n == 0) return CHPL_OK;
    const Plan p = plan(*a);
    CHPL_TRY(chpl::linear::check_work("mx4_linear", work, work_bytes, p.bytes));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    chpl_mx4 x = a->x4;
    if (p.bytes) {
        x.codes = static_cast<uint8_t*>(work);
        x.scales = x.codes + p.scales;
        x.ldc = code_bytes(a->k);
        CHPL_TRY(pack(st, a->type, a->tokens, a->k, a->x, a->ldx, x));
    }
    chpl::linear::Epilogue e = {};
    e.m = (int)a->n;
    e.n = (int)a->tokens;
    e.act = a->act;
    e.out = a->y;
    e.ldo = a->ldy;
    e.bias = a->bias;
    e.add = a->residual;
    e.ldadd = a->ldr;
    return gemm(st, a->type, a->w4, x, a->k, e);
}
