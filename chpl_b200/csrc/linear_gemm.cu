// The linear-layer products: D[f][t] = sum_c A(f, c) B(t, c) with the
// epilogue of linear_epilogue.cuh.
//
// Every product is oriented so that the output's contiguous dimension is f,
// the dimension that a warp's lanes run along when they store.
#include "linear_epilogue.cuh"

namespace chpl {
namespace linear {

__device__ int g_status;  // sticky device-side error of this module

constexpr int TF = 128, TT = 32, TC = 32;

// FP32 multiply-adds from shared memory: a thread per feature, 32 rows each
template <typename T, Kind KIND>
__global__ void __launch_bounds__(TF) simple_kernel(const T* __restrict__ A, int64_t lda, bool akm,
                                                    const T* __restrict__ B, int64_t ldb, bool bkm, int k, Epilogue e)
{
    __shared__ float sa[TC][TF + 1];
    __shared__ float sb[TC][TT + 4];
    const int f0 = blockIdx.x * TF, t0 = blockIdx.y * TT, tid = threadIdx.x;
    float acc[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[j] = 0.0f;
    for (int c0 = 0; c0 < k; c0 += TC) {
        for (int i = tid; i < TF * TC; i += TF) {
            const int c = akm ? i % TC : i / TF, f = akm ? i / TC : i % TF;
            const bool in = f0 + f < e.m && c0 + c < k;
            sa[c][f] = in ? to_f32(akm ? A[(int64_t)(f0 + f) * lda + c0 + c] : A[(int64_t)(c0 + c) * lda + f0 + f]) : 0.0f;
        }
        for (int i = tid; i < TT * TC; i += TF) {
            const int c = bkm ? i % TC : i / TT, t = bkm ? i / TC : i % TT;
            const bool in = t0 + t < e.n && c0 + c < k;
            sb[c][t] = in ? to_f32(bkm ? B[(int64_t)(t0 + t) * ldb + c0 + c] : B[(int64_t)(c0 + c) * ldb + t0 + t]) : 0.0f;
        }
        __syncthreads();
#pragma unroll 4
        for (int c = 0; c < TC; ++c) {
            const float a = sa[c][tid];
#pragma unroll
            for (int j = 0; j < TT; ++j) acc[j] = fmaf(a, sb[c][j], acc[j]);
        }
        __syncthreads();
    }
    epilogue<T, KIND, TT>(e, f0 + tid, t0, acc, bias_of<T>(e, f0 + tid));
}

template <typename T, Kind KIND>
static int launch(cudaStream_t st, const Operand& a, const Operand& b, int64_t k, const Epilogue& e)
{
    for (int64_t t = 0; t < e.n; t += (int64_t)65535 * TT) {  // the grid's second dimension ends at 65535
        const int64_t nt = e.n - t < (int64_t)65535 * TT ? e.n - t : (int64_t)65535 * TT;
        if (t != 0) { set_error("linear: more than %d rows", 65535 * TT); return CHPL_ERR_UNSUPPORTED; }
        const dim3 grid((unsigned)((e.m + TF - 1) / TF), (unsigned)((nt + TT - 1) / TT));
        simple_kernel<T, KIND><<<grid, TF, 0, st>>>(static_cast<const T*>(a.p), a.ld, a.k_major,
                                                    static_cast<const T*>(b.p), b.ld, b.k_major, (int)k, e);
        CHPL_CUDA(cudaGetLastError());
    }
    return CHPL_OK;
}

template <typename T>
static int launch_kind(cudaStream_t st, Kind kind, const Operand& a, const Operand& b, int64_t k, const Epilogue& e)
{
    if (kind == kForward) return launch<T, kForward>(st, a, b, k, e);
    if (kind == kGradInput) return launch<T, kGradInput>(st, a, b, k, e);
    return launch<T, kGradWeight>(st, a, b, k, e);
}

int gemm(cudaStream_t st, int type, Kind kind, const Operand& a, const Operand& b, int64_t k, const Epilogue& e)
{
    if (e.m == 0 || e.n == 0) return CHPL_OK;
    return type == CHPL_TYPE_BF16 ? launch_kind<__nv_bfloat16>(st, kind, a, b, k, e)
                                  : launch_kind<__half>(st, kind, a, b, k, e);
}

int read_clear_status(int* st)
{
    int v = 0, z = 0;
    CHPL_CUDA(cudaMemcpyFromSymbol(&v, g_status, sizeof(int)));
    CHPL_CUDA(cudaMemcpyToSymbol(g_status, &z, sizeof(int)));
    *st = v;
    return CHPL_OK;
}

}  // namespace linear
}  // namespace chpl
