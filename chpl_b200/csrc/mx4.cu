// Microscaled 4-bit floating point (OCP MXFP4): pack and unpack, and the C entry
// points chpl_mx4_pack, chpl_mx4_unpack and chpl_mx4_linear.
//
// Bound: HBM.  A matrix of T x D elements of e bytes moves e T D + T D (1 / 2 +
// 1 / 32) bytes each way.
#include <algorithm>

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

// A warp takes UNITS x 256 columns of a row at a time, a lane eight consecutive
// ones of each, every load before any arithmetic.  A group is four lanes; the
// scales of a block, four groups, are a word in memory, which the lanes' scales of
// all units are turned about into at once.  8192 x 16384 BF16: 61 us, 5.6 TB/s (98
// with a word put together and placed for each unit); issue slots 73 % busy.
template <typename T, int UNITS>
__global__ void __launch_bounds__(kRowsThreads) pack_kernel(const RowsIn<T> in, const chpl_mx4 c, const int64_t items, const uint32_t segs,
                                                            const int cols)
{
    start_of_inputs();
    const int lane = lane_id(), groups_end = (cols + kGroup - 1) / kGroup * kGroup;
    const int64_t blocks = blocks_of(cols), step = (int64_t)gridDim.x * (kRowsThreads / 32);
    for (int64_t i = (int64_t)blockIdx.x * (kRowsThreads / 32) + warp_id(); i < items; i += step) {
        const uint32_t t = items < 0xffffffffll ? (uint32_t)i / segs : (uint32_t)(i / segs);
        const int seg = (int)(i - (int64_t)t * segs), j0 = seg * (UNITS * kPiece) + lane * 8;
        typename RowsIn<T>::Raw raw[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) raw[u] = in.raw(t, j0 + u * kPiece, cols);
        uint8_t* codes = c.codes + (int64_t)t * c.ldc + j0 / 2;
        uint32_t scales = 0;  // of the lane's group in each unit
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            float v[8];
            in.value(raw[u], v);
            uint32_t top = in.top(raw[u]);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t s = scale_of(top);
            uint32_t w = codes8(v, inv_step(s));
            if (s == kBadScale) w = 0;
            if (j0 + u * kPiece < groups_end) *reinterpret_cast<uint32_t*>(codes + u * (kPiece / 2)) = w;
            scales |= s << (8 * u);
        }
        // lane 2 u + h: the four groups of half h of unit u
        uint32_t g[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) g[q] = __shfl_sync(0xffffffffu, scales, 16 * (lane & 1) + 4 * q);
        const int u = lane / 2 % UNITS, block = seg * (2 * UNITS) + lane;
        const uint32_t lo = __byte_perm(g[0], g[1], u | (4 + u) << 4), hi = __byte_perm(g[2], g[3], u | (4 + u) << 4);
        if (lane < 2 * UNITS && block < blocks) *reinterpret_cast<uint32_t*>(c.scales + scale_at(t, block, blocks)) = __byte_perm(lo, hi, 0x5410);
    }
}

// The way back, in the same pieces: the words of scales of all units are read by
// eight lanes and dealt out (8192 x 16384 to BF16: 62 us; 66 with a byte read for
// each lane and unit).
template <typename T, int UNITS>
__global__ void __launch_bounds__(kRowsThreads) unpack_kernel(const chpl_mx4 c, const RowsOut<T> out, const int64_t items, const uint32_t segs,
                                                              const int cols)
{
    __shared__ uint4 turns[kRowsThreads / 32][64];  // 256 elements of up to 4 bytes for each warp
    start_of_inputs();
    const int lane = lane_id();
    const int64_t blocks = blocks_of(cols), step_items = (int64_t)gridDim.x * (kRowsThreads / 32);
    for (int64_t i = (int64_t)blockIdx.x * (kRowsThreads / 32) + warp_id(); i < items; i += step_items) {
        const uint32_t t = items < 0xffffffffll ? (uint32_t)i / segs : (uint32_t)(i / segs);
        const int seg = (int)(i - (int64_t)t * segs), j0 = seg * (UNITS * kPiece) + lane * 8, block = seg * (2 * UNITS) + lane;
        const uint8_t* codes = c.codes + (int64_t)t * c.ldc + j0 / 2;
        uint32_t w[UNITS], four = 0;  // lane 2 u + h: the four scales of half h of unit u
#pragma unroll
        for (int u = 0; u < UNITS; ++u) w[u] = j0 + u * kPiece < cols ? __ldg(reinterpret_cast<const uint32_t*>(codes + u * (kPiece / 2))) : 0;
        if (lane < 2 * UNITS && block < blocks) four = __ldg(reinterpret_cast<const uint32_t*>(c.scales + scale_at(t, block, blocks)));
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t s = __shfl_sync(0xffffffffu, four, 2 * u + (lane >> 4)) >> (lane >> 2 & 3) * 8 & 0xffu;
            float v[8];
            values8(w[u], step(s), v);
            out.put_warp(t, j0 + u * kPiece, cols, v, turns[warp_id()]);
        }
    }
}

// A launch over `rows` rows, in pieces of four units where rows are long and that
// leaves every warp a piece, else of one
template <typename L>
static int in_pieces(int64_t rows, int64_t cols, L&& launch)
{
    constexpr int64_t kWarps = kRowsThreads / 32, kBlocks = 148 * 8;  // eight resident blocks per SM, then a grid stride
    const int units = cols > kPiece && rows * ((cols + 4 * kPiece - 1) / (4 * kPiece)) >= kBlocks * kWarps ? 4 : 1;
    const int64_t segs = (cols + units * kPiece - 1) / (units * kPiece), items = rows * segs;
    return launch(units, std::min((items + kWarps - 1) / kWarps, kBlocks), items, (uint32_t)segs);
}

template <typename T>
static int pack(cudaStream_t st, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4& c)
{
    return in_pieces(rows, cols, [&](int units, int64_t blocks, int64_t items, uint32_t segs) {
        return launch_kernel(units == 4 ? pack_kernel<T, 4> : pack_kernel<T, 1>, blocks, kRowsThreads, 0, 1, st, rows_in<T>(x, ldx), c, items, segs, (int)cols);
    });
}

template <typename T>
static int unpack(cudaStream_t st, int64_t rows, int64_t cols, void* x, int64_t ldx, const chpl_mx4& c)
{
    return in_pieces(rows, cols, [&](int units, int64_t blocks, int64_t items, uint32_t segs) {
        return launch_kernel(units == 4 ? unpack_kernel<T, 4> : unpack_kernel<T, 1>, blocks, kRowsThreads, 0, 1, st, c, rows_out<T>(x, ldx), items, segs,
                             (int)cols);
    });
}

int pack(cudaStream_t st, int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const chpl_mx4& c)
{
    if (type == CHPL_TYPE_BF16) return pack<__nv_bfloat16>(st, rows, cols, x, ldx, c);
    if (type == CHPL_TYPE_F16) return pack<__half>(st, rows, cols, x, ldx, c);
    return pack<float>(st, rows, cols, x, ldx, c);
}

// the workspace: codes and scales of X, where it comes in 16 bits and is coded first
struct CodedInput {
    size_t scales = 0, bytes = 0;
};

static CodedInput coded_input(const chpl_mx4_fwd& a)
{
    CodedInput p;
    if (a.x4.codes || a.tokens <= kCodedRows || a.n == 0 || a.k == 0) return p;
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
    *work_bytes = coded_input(*a).bytes;
    return CHPL_OK;
}

extern "C" int chpl_mx4_linear(void* stream, const chpl_mx4_fwd* a, void* work, size_t work_bytes)
{
    using namespace chpl::mx4;
    CHPL_TRY(check("mx4_linear", a, true));
    if (a->tokens == 0 || a->n == 0) return CHPL_OK;
    const CodedInput p = coded_input(*a);
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
    return gemm(st, a->type, a->w4, x, x.codes || a->k == 0 ? nullptr : a->x, a->ldx, a->k, e);
}
