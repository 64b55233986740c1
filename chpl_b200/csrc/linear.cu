// Linear layers of a model: argument checks, workspace layout, the elementwise
// kernels around the products, and the C entry points chpl_linear_forward /
// chpl_linear_backward.
//
// Forward: one product.  Backward: G = dY * act'(Z) and its column sums (one
// pass over dY and Z), the layer's input out of its checkpoint, then the two
// products dX = G W and dW = G^T Xv.
#include "linear.h"

#include <algorithm>
#include <type_traits>

#include "linear_epilogue.cuh"

namespace chpl {
namespace linear {

// ----------------------------------------------------------------------------
// checks
// ----------------------------------------------------------------------------
int check_size(const char* who, const char* what, int64_t v)
{
    if (v < 0) { set_error("%s: %s = %lld is negative", who, what, (long long)v); return CHPL_ERR_INVALID; }
    if (v > kMaxSize) { set_error("%s: %s = %lld exceeds %lld", who, what, (long long)v, (long long)kMaxSize); return CHPL_ERR_UNSUPPORTED; }
    return CHPL_OK;
}

int check_operand(const char* who, const char* what, const void* p, int64_t ld, int64_t width, int elt)
{
    if (!p) { set_error("%s: %s is NULL", who, what); return CHPL_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(p) % elt) { set_error("%s: %s is not aligned to its elements", who, what); return CHPL_ERR_INVALID; }
    if (ld < width) { set_error("%s: row distance of %s is %lld, below its %lld columns", who, what, (long long)ld, (long long)width); return CHPL_ERR_INVALID; }
    if (ld > kMaxLd) { set_error("%s: row distance of %s is %lld, above %lld", who, what, (long long)ld, (long long)kMaxLd); return CHPL_ERR_UNSUPPORTED; }
    return CHPL_OK;
}

int check_ckpt(const char* who, const char* what, const chpl_ckpt8& c, int64_t width)
{
    CHPL_TRY(check_operand(who, what, c.codes, c.ldc, width, 1));
    return check_operand(who, "its scales", c.scales, c.lds, (width + kCkptGroup - 1) / kCkptGroup, 1);
}

static int check_type(const char* who, int type)
{
    if (type == CHPL_TYPE_BF16 || type == CHPL_TYPE_F16) return CHPL_OK;
    set_error("%s: type %d is not BF16 or F16", who, type);
    return CHPL_ERR_INVALID;
}

static int check_act(const char* who, int act)
{
    if (act >= CHPL_ACT_NONE && act <= CHPL_ACT_SILU) return CHPL_OK;
    set_error("%s: unknown activation %d", who, act);
    return CHPL_ERR_INVALID;
}

int check_work(const char* who, const void* work, size_t have, size_t need)
{
    if (have < need || (need && !work)) { set_error("%s: workspace of %zu bytes, %zu are needed", who, work ? have : (size_t)0, need); return CHPL_ERR_WORKSPACE; }
    if (need && reinterpret_cast<uintptr_t>(work) % 256) { set_error("%s: workspace is not 256-byte aligned", who); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

// ----------------------------------------------------------------------------
// elementwise kernels
// ----------------------------------------------------------------------------
struct Activate {
    int act;
    __device__ __forceinline__ void operator()(float (&v)[8]) const
    {
        with_act(act, [&](auto tag) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) activate<decltype(tag)::value>(v[i], v[i + 1]);
        });
    }
};

// A layer's incoming gradient: G = dY * act'(Z) into g (where given), and the
// sums of its columns.  One pass over dY and Z: HBM-bound.
//
// A block takes 256 columns (a lane 8 consecutive ones) of one chunk of rows,
// its warps every eighth row of it.  Up to 1024 tokens are eight chunks, the
// blocks of a cluster, which joins their sums in shared memory: one launch does
// it (257 x 519: 6 us; two launches with chunks of 128 rows 18).  More tokens
// leave each chunk's sums in part[chunk][n], which sum_chunks_kernel adds
// (8192 x 16384: 50 us, 5.3 TB/s; in clusters 104).  Every order is fixed.
constexpr int kSumThreads = 256;
constexpr int kSumWarps = kSumThreads / 32;
constexpr int kSumCluster = 8;

struct SumShape {
    int rows;     // of a chunk
    int chunks;
    int cluster;  // blocks that join their sums: 1 or kSumCluster
};

// chunks of 128 rows where that makes four blocks per SM, else of 64
static SumShape sum_shape(int64_t tokens, int64_t n)
{
    if (tokens <= 128 * kSumCluster)
        return {(int)round_up((size_t)(tokens + kSumCluster - 1) / kSumCluster, kSumWarps), tokens > 0 ? 1 : 0, kSumCluster};
    const int rows = (tokens + 127) / 128 * ((n + 255) / 256) >= 4 * 148 ? 128 : 64;
    return {rows, (int)((tokens + rows - 1) / rows), 1};
}

// db, of the operands' type T or FP32
struct Sums {
    void* db;
    int f32, accumulate;
};

template <typename T>
__device__ __forceinline__ void put_sum(const Sums& s, int j, float v)
{
    if (s.f32) {
        float* o = static_cast<float*>(s.db) + j;
        *o = s.accumulate ? *o + v : v;
    } else {
        T* o = static_cast<T*>(s.db) + j;
        *o = from_f32<T>(s.accumulate ? to_f32(*o) + v : v);
    }
}

struct NoZ {
    struct Raw {};
    __device__ __forceinline__ Raw raw(int64_t, int, int) const { return {}; }
    __device__ __forceinline__ void value(const Raw&, float (&)[8]) const {}
};

template <typename T, typename Z>
__global__ void __launch_bounds__(kSumThreads) grad_act_kernel(RowsIn<T> dy, Z z, int act, int rows, int n, int chunk_rows,
                                                               int cluster, RowsOut<T> g, float* __restrict__ part, Sums out)
{
    constexpr int kAhead = std::is_same<Z, NoZ>::value ? 4 : 2;  // rows whose loads are under way at once
    __shared__ float sums[kSumWarps][256 + 8];
    const int blocks = (n + 255) / 256, cl = blockIdx.x / cluster, rank = blockIdx.x - cl * cluster;
    const int group = cl / blocks, j0 = (cl - group * blocks) * 256;
    const int lane = lane_id(), warp = warp_id(), j = j0 + lane * 8;
    const int64_t first = ((int64_t)group * cluster + rank) * chunk_rows;
    const int count = (int)max((int64_t)0, min((int64_t)chunk_rows, rows - first));
    float sum[8] = {};
    start_of_inputs();
    for (int r = warp; r < count; r += kAhead * kSumWarps) {
        typename RowsIn<T>::Raw a[kAhead];
        typename Z::Raw b[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (r + u * kSumWarps < count) {
                a[u] = dy.raw(first + r + u * kSumWarps, j, n);
                b[u] = z.raw(first + r + u * kSumWarps, j, n);
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (r + u * kSumWarps < count) {
                float v[8];
                dy.value(a[u], v);
                if (!std::is_same<Z, NoZ>::value) {
                    float zv[8];
                    z.value(b[u], zv);
                    with_act(act, [&](auto tag) {
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            float sa, sb;
                            slope_and_value<decltype(tag)::value>(zv[i], zv[i + 1], sa, sb);
                            v[i] *= sa;
                            v[i + 1] *= sb;
                        }
                    });
                }
                if (g.p) g.put(first + r + u * kSumWarps, j, n, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += v[i];
            }
    }
    if (!out.db) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    const int c = threadIdx.x;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kSumWarps; ++w) total += sums[w][c];
    if (cluster == 1) {
        if (j0 + c < n) part[(int64_t)group * n + j0 + c] = total;
        return;
    }
    __syncthreads();
    sums[0][c] = total;
    cluster_sync();
    if (c < 256 / kSumCluster) {  // block r adds up the columns r 32 .. r 32 + 31
        const int at = rank * (256 / kSumCluster) + c;
        total = 0.0f;
#pragma unroll
        for (int r = 0; r < kSumCluster; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(smem_u32(&sums[0][at]), (uint32_t)r)) : "memory");
            total += v;
        }
        if (j0 + at < n) put_sum<T>(out, j0 + at, total);
    }
    cluster_sync();  // no block leaves while another still reads its sums
}

// db[j] (+)= sum of part[0..chunks)[j].  A block takes 32 columns, its warps (one
// for every 32 chunks) equal runs of the chunks, and the runs' sums are joined in
// order.  Bound by the loads' latency: db of 100000 x 256, 1563 chunks, 16 us with
// its first pass, a million x 128 130 us, where a thread for a whole column took 55
// and 520; dX's sum on top of dX of 8192 x 128, 1024 parts, 3 us (32).
constexpr int kJoinWarps = 32;

static int join_warps(int64_t chunks) { return (int)std::max<int64_t>(1, std::min<int64_t>(kJoinWarps, chunks / 32)); }

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) sum_chunks_kernel(const float* __restrict__ part, int chunks, int n, Sums out)
{
    __shared__ float sums[kJoinWarps][32];
    const int lane = lane_id(), warp = warp_id(), warps = blockDim.x / 32, j = blockIdx.x * 32 + lane;
    const int first = (int)((int64_t)chunks * warp / warps), last = (int)((int64_t)chunks * (warp + 1) / warps);
    start_of_inputs();
    float sum = 0.0f;
    if (j < n) {
#pragma unroll 8
        for (int ch = first; ch < last; ++ch) sum += part[(int64_t)ch * n + j];
    }
    if (warps > 1) {
        sums[warp][lane] = sum;
        __syncthreads();
        if (warp > 0) return;
        for (int w = 1; w < warps; ++w) sum += sums[w][lane];
    }
    if (j < n) put_sum<T>(out, j, sum);
}

// launches it
template <typename T>
static int join_sums(cudaStream_t st, const float* part, int64_t chunks, int64_t n, const Sums& out)
{
    return launch_kernel(sum_chunks_kernel<T>, (n + 31) / 32, 32 * join_warps(chunks), 0, 1, st, part, (int)chunks, (int)n, out);
}

// ----------------------------------------------------------------------------
// layout
// ----------------------------------------------------------------------------
// TMA reads rows whose base and distance are multiples of 16 bytes; a single
// row has no distance
static bool tma_rows(const void* p, int64_t ld, int64_t rows)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || ld % 8 == 0);
}

static int64_t padded(int64_t width) { return (int64_t)round_up((size_t)width, 8); }

struct Arena {
    size_t used = 0;
    size_t take(size_t bytes)
    {
        const size_t at = used;
        used += round_up(bytes, 256);
        return at;
    }
};

// A 16-bit matrix as a product reads it: in place, or at `at` in the workspace
struct Staged {
    bool copy = false;
    size_t at = 0;
    int64_t ld = 0;
};

static Staged stage(Arena& a, bool copy, int64_t ld, int64_t rows, int64_t cols)
{
    Staged s;
    s.copy = copy;
    s.ld = copy || rows <= 1 ? padded(cols) : ld;
    if (copy) s.at = a.take((size_t)rows * s.ld * 2);
    return s;
}

static const void* at(const Staged& s, const void* in_place, void* work)
{
    return s.copy ? static_cast<char*>(work) + s.at : in_place;
}

struct ForwardPlan {
    Staged x, w;
    size_t bytes;
};

static ForwardPlan plan(const chpl_linear_fwd& a)
{
    Arena m;
    ForwardPlan p;
    const bool any = a.tokens > 0 && a.n > 0 && a.k > 0;
    p.x = stage(m, any && !tma_rows(a.x, a.ldx, a.tokens), a.ldx, a.tokens, a.k);
    p.w = stage(m, any && !tma_rows(a.w, a.ldw, a.n), a.ldw, a.n, a.k);
    p.bytes = m.used;
    return p;
}

struct BackwardPlan {
    Staged g, w, x;
    bool need_xv;   // Xv is not X as it stands
    size_t part;
    size_t sums;    // of dX's columns
    SumShape sum;   // of db
    size_t bytes;
};

static BackwardPlan plan(const chpl_linear_bwd& a)
{
    Arena m;
    BackwardPlan p;
    const bool any = a.tokens > 0 && a.n > 0;
    const bool products = any && (a.dx || a.dw) && a.k > 0;
    p.g = stage(m, products && (a.act != CHPL_ACT_NONE || !tma_rows(a.dy, a.lddy, a.tokens)), a.lddy, a.tokens, a.n);
    p.w = stage(m, products && a.dx && !tma_rows(a.w, a.ldw, a.n), a.ldw, a.n, a.k);
    p.need_xv = a.x8.codes || a.in_act != CHPL_ACT_NONE || !tma_rows(a.x, a.ldx, a.tokens);
    p.x = stage(m, products && a.dw && p.need_xv, a.ldx, a.tokens, a.k);
    p.sum = sum_shape(a.tokens, a.n);
    p.part = a.db && a.n > 0 && p.sum.cluster == 1 ? m.take((size_t)p.sum.chunks * a.n * 4) : 0;
    p.sums = a.dx_sum && a.k > 0 ? m.take((size_t)sum_parts(a.k, a.tokens, a.n) * a.k * 4) : 0;
    p.bytes = m.used;
    return p;
}

static int check(const char* who, const chpl_linear_fwd* a, bool pointers)
{
    if (!a) { set_error("%s: arguments are NULL", who); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_type(who, a->type));
    CHPL_TRY(check_act(who, a->act));
    CHPL_TRY(check_size(who, "tokens", a->tokens));
    CHPL_TRY(check_size(who, "n", a->n));
    CHPL_TRY(check_size(who, "k", a->k));
    if (!pointers || a->tokens == 0 || a->n == 0) return CHPL_OK;
    if (a->k > 0) {
        CHPL_TRY(check_operand(who, "x", a->x, a->ldx, a->k, 2));
        CHPL_TRY(check_operand(who, "w", a->w, a->ldw, a->k, 2));
    }
    CHPL_TRY(check_operand(who, "y", a->y, a->ldy, a->n, 2));
    if (a->bias) CHPL_TRY(check_operand(who, "bias", a->bias, a->n, a->n, 2));
    if (a->residual) CHPL_TRY(check_operand(who, "residual", a->residual, a->ldr, a->n, 2));
    if (a->z) CHPL_TRY(check_operand(who, "z", a->z, a->ldz, a->n, 2));
    if (a->z8.codes) CHPL_TRY(check_ckpt(who, "z8", a->z8, a->n));
    if (a->y == a->residual && a->ldy != a->ldr) { set_error("%s: y is residual with another row distance", who); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

static int check(const char* who, const chpl_linear_bwd* a, bool pointers)
{
    if (!a) { set_error("%s: arguments are NULL", who); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_type(who, a->type));
    CHPL_TRY(check_act(who, a->act));
    CHPL_TRY(check_act(who, a->in_act));
    if (a->grad_type != a->type && a->grad_type != CHPL_TYPE_F32) {
        set_error("%s: grad_type %d is neither the operands' type nor F32", who, a->grad_type);
        return CHPL_ERR_INVALID;
    }
    CHPL_TRY(check_size(who, "tokens", a->tokens));
    CHPL_TRY(check_size(who, "n", a->n));
    CHPL_TRY(check_size(who, "k", a->k));
    if (!pointers) return CHPL_OK;
    const int ge = a->grad_type == CHPL_TYPE_F32 ? 4 : 2;
    if (a->dx && a->tokens > 0 && a->k > 0) {
        CHPL_TRY(check_operand(who, "dx", a->dx, a->lddx, a->k, 2));
        if (a->n > 0) CHPL_TRY(check_operand(who, "w", a->w, a->ldw, a->k, 2));
        if (a->add) CHPL_TRY(check_operand(who, "add", a->add, a->ldadd, a->k, 2));
        if (a->dx == a->add && a->lddx != a->ldadd) { set_error("%s: dx is add with another row distance", who); return CHPL_ERR_INVALID; }
    }
    if (a->dw && a->n > 0 && a->k > 0) CHPL_TRY(check_operand(who, "dw", a->dw, a->lddw, a->k, ge));
    if (a->db && a->n > 0) CHPL_TRY(check_operand(who, "db", a->db, a->n, a->n, ge));
    if (a->dx_sum && a->k > 0) CHPL_TRY(check_operand(who, "dx_sum", a->dx_sum, a->k, a->k, ge));
    if (a->dx_sum && !a->dx && a->tokens > 0 && a->k > 0) { set_error("%s: dx_sum without dx", who); return CHPL_ERR_INVALID; }
    const bool any = a->tokens > 0 && a->n > 0 && (a->dx || a->dw || a->db);
    if (any) {
        CHPL_TRY(check_operand(who, "dy", a->dy, a->lddy, a->n, 2));
        if (a->act != CHPL_ACT_NONE) {
            if (a->z8.codes) CHPL_TRY(check_ckpt(who, "z8", a->z8, a->n));
            else CHPL_TRY(check_operand(who, "z", a->z, a->ldz, a->n, 2));
        }
    }
    // dW's operand; with in_act dX's epilogue reads it, of outputs of the layer or of none (n = 0)
    if (a->tokens > 0 && a->k > 0 && ((a->dw && a->n > 0) || (a->dx && a->in_act != CHPL_ACT_NONE))) {
        if (a->x8.codes) CHPL_TRY(check_ckpt(who, "x8", a->x8, a->k));
        else CHPL_TRY(check_operand(who, "x", a->x, a->ldx, a->k, 2));
    }
    return CHPL_OK;
}

// ----------------------------------------------------------------------------
// the two passes
// ----------------------------------------------------------------------------
// An operand of a product as TMA can read it: the values of a checkpoint, an
// activation of either, or a copy.
template <typename T>
using CkptJob = RowsJob<CkptIn, RowsOut<T>, Activate>;
template <typename T>
using CopyJob = RowsJob<RowsIn<T>, RowsOut<T>, Activate>;

template <typename T>
static CopyJob<T> copy_job(const void* x, int64_t ldx, int act, int64_t rows, int64_t cols, void* out, int64_t ldo)
{
    return CopyJob<T>(rows_in<T>(x, ldx), rows_out<T>(out, ldo), Activate{act}, rows, cols);
}

template <typename T>
static CkptJob<T> ckpt_job(const chpl_ckpt8& c, int act, int64_t rows, int64_t cols, void* out, int64_t ldo)
{
    return CkptJob<T>(ckpt_in(c), rows_out<T>(out, ldo), Activate{act}, rows, cols);
}

template <typename T>
static int forward(cudaStream_t st, const chpl_linear_fwd& a, void* work)
{
    const ForwardPlan p = plan(a);
    char* wk = static_cast<char*>(work);
    const auto xj = [&] { return copy_job<T>(a.x, a.ldx, CHPL_ACT_NONE, a.tokens, a.k, wk + p.x.at, p.x.ld); };
    const auto wj = [&] { return copy_job<T>(a.w, a.ldw, CHPL_ACT_NONE, a.n, a.k, wk + p.w.at, p.w.ld); };
    if (p.x.copy && p.w.copy) CHPL_TRY(run_rows(st, xj(), wj()));
    else if (p.x.copy) CHPL_TRY(run_rows(st, xj()));
    else if (p.w.copy) CHPL_TRY(run_rows(st, wj()));
    Epilogue e = {};
    e.m = (int)a.n;
    e.n = (int)a.tokens;
    e.act = a.act;
    e.out = a.y;
    e.ldo = a.ldy;
    e.bias = a.bias;
    e.add = a.residual;
    e.ldadd = a.ldr;
    e.z = a.z;
    e.ldz = a.ldz;
    e.z8 = a.z8;
    return gemm(st, a.type, kForward, {at(p.w, a.w, work), p.w.ld, true}, {at(p.x, a.x, work), p.x.ld, true}, a.k, e);
}

template <typename T>
static int backward(cudaStream_t st, const chpl_linear_bwd& a, void* work)
{
    const BackwardPlan p = plan(a);
    char* wk = static_cast<char*>(work);
    if (a.n > 0 && (p.g.copy || a.db)) {
        const Sums sums = {a.db, a.grad_type == CHPL_TYPE_F32, a.accumulate};
        // one cluster's sums go straight to db, chunks' (or none: zeros) by way of the workspace
        const bool join = a.db && (p.sum.cluster == 1 || a.tokens == 0);
        float* part = join ? reinterpret_cast<float*>(wk + p.part) : nullptr;
        if (a.tokens > 0) {
            const int64_t blocks = (a.n + 255) / 256 * (int64_t)p.sum.chunks * p.sum.cluster;
            if (blocks > 0x7fffffff) { set_error("linear_backward: dy of %lld x %lld is more than one launch serves", (long long)a.tokens, (long long)a.n); return CHPL_ERR_UNSUPPORTED; }
            const RowsIn<T> dy = rows_in<T>(a.dy, a.lddy);
            const RowsOut<T> go = rows_out<T>(p.g.copy ? wk + p.g.at : nullptr, p.g.ld);
            const int rows = (int)a.tokens, n = (int)a.n;
            if (a.act == CHPL_ACT_NONE)
                CHPL_TRY(launch_kernel(grad_act_kernel<T, NoZ>, blocks, kSumThreads, 0, p.sum.cluster, st, dy, NoZ(), a.act, rows, n, p.sum.rows,
                                       p.sum.cluster, go, part, sums));
            else if (a.z8.codes)
                CHPL_TRY(launch_kernel(grad_act_kernel<T, CkptIn>, blocks, kSumThreads, 0, p.sum.cluster, st, dy, ckpt_in(a.z8), a.act, rows, n,
                                       p.sum.rows,
                                       p.sum.cluster, go, part, sums));
            else
                CHPL_TRY(launch_kernel(grad_act_kernel<T, RowsIn<T>>, blocks, kSumThreads, 0, p.sum.cluster, st, dy, rows_in<T>(a.z, a.ldz), a.act,
                                       rows, n, p.sum.rows,
                                       p.sum.cluster, go, part, sums));
        }
        if (join) CHPL_TRY(join_sums<T>(st, part, p.sum.chunks, a.n, sums));
    }
    if (a.k == 0) return CHPL_OK;
    const Operand g_rows = {at(p.g, a.dy, work), p.g.ld, true}, g_cols = {g_rows.p, p.g.ld, false};
    // an activation's value comes with its slope out of dX's epilogue
    const bool xv_from_dx = p.x.copy && a.dx && a.in_act != CHPL_ACT_NONE;
    const bool expand = p.x.copy && !xv_from_dx;
    const auto wj = [&] { return copy_job<T>(a.w, a.ldw, CHPL_ACT_NONE, a.n, a.k, wk + p.w.at, p.w.ld); };
    if (expand && a.x8.codes) {
        const CkptJob<T> xj = ckpt_job<T>(a.x8, a.in_act, a.tokens, a.k, wk + p.x.at, p.x.ld);
        CHPL_TRY(p.w.copy ? run_rows(st, xj, wj()) : run_rows(st, xj));
    } else if (expand) {
        const CopyJob<T> xj = copy_job<T>(a.x, a.ldx, a.in_act, a.tokens, a.k, wk + p.x.at, p.x.ld);
        CHPL_TRY(p.w.copy ? run_rows(st, xj, wj()) : run_rows(st, xj));
    } else if (p.w.copy) {
        CHPL_TRY(run_rows(st, wj()));
    }
    if (a.dx) {
        Epilogue e = {};
        e.m = (int)a.k;
        e.n = (int)a.tokens;
        e.act = a.in_act;
        e.out = a.dx;
        e.ldo = a.lddx;
        e.add = a.add;
        e.ldadd = a.ldadd;
        e.z = const_cast<void*>(a.x);
        e.ldz = a.ldx;
        e.z8 = a.x8;
        e.xv = xv_from_dx ? wk + p.x.at : nullptr;
        e.ldxv = p.x.ld;
        e.sums = a.dx_sum ? reinterpret_cast<float*>(wk + p.sums) : nullptr;
        CHPL_TRY(gemm(st, a.type, kGradInput, {at(p.w, a.w, work), p.w.ld, false}, g_rows, a.n, e));
    }
    if (a.dx_sum)
        CHPL_TRY(join_sums<T>(st, reinterpret_cast<const float*>(wk + p.sums), sum_parts(a.k, a.tokens, a.n), a.k,
                              Sums{a.dx_sum, a.grad_type == CHPL_TYPE_F32, a.accumulate}));
    if (a.dw && (a.tokens > 0 || !a.accumulate)) {
        Epilogue e = {};
        e.m = (int)a.k;
        e.n = (int)a.n;
        e.out_f32 = a.grad_type == CHPL_TYPE_F32;
        e.out = a.dw;
        e.ldo = a.lddw;
        e.add = a.accumulate ? a.dw : nullptr;
        e.ldadd = a.lddw;
        CHPL_TRY(gemm(st, a.type, kGradWeight, {at(p.x, a.x, work), p.x.ld, false}, g_cols, a.tokens, e));
    }
    return CHPL_OK;
}

}  // namespace linear
}  // namespace chpl

extern "C" int chpl_linear_forward_worksize(const chpl_linear_fwd* a, size_t* work_bytes)
{
    using namespace chpl::linear;
    CHPL_TRY(check("linear_forward_worksize", a, false));
    if (!work_bytes) { chpl::set_error("linear_forward_worksize: work_bytes is NULL"); return CHPL_ERR_INVALID; }
    *work_bytes = plan(*a).bytes;
    return CHPL_OK;
}

extern "C" int chpl_linear_forward(void* stream, const chpl_linear_fwd* a, void* work, size_t work_bytes)
{
    using namespace chpl::linear;
    CHPL_TRY(check("linear_forward", a, true));
    if (a->tokens == 0 || a->n == 0) return CHPL_OK;
    CHPL_TRY(check_work("linear_forward", work, work_bytes, plan(*a).bytes));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->type == CHPL_TYPE_BF16 ? forward<__nv_bfloat16>(st, *a, work) : forward<__half>(st, *a, work);
}

extern "C" int chpl_linear_backward_worksize(const chpl_linear_bwd* a, size_t* work_bytes)
{
    using namespace chpl::linear;
    CHPL_TRY(check("linear_backward_worksize", a, false));
    if (!work_bytes) { chpl::set_error("linear_backward_worksize: work_bytes is NULL"); return CHPL_ERR_INVALID; }
    *work_bytes = plan(*a).bytes;
    return CHPL_OK;
}

extern "C" int chpl_linear_backward(void* stream, const chpl_linear_bwd* a, void* work, size_t work_bytes)
{
    using namespace chpl::linear;
    CHPL_TRY(check("linear_backward", a, true));
    CHPL_TRY(check_work("linear_backward", work, work_bytes, plan(*a).bytes));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->type == CHPL_TYPE_BF16 ? backward<__nv_bfloat16>(st, *a, work) : backward<__half>(st, *a, work);
}
