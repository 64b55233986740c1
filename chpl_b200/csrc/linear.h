// Internal interface of the linear-layer module (linear.cu, linear_gemm.cu, ckpt8.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "chpl.h"

namespace chpl {
namespace linear {

// Sizes fit the kernels' int32 coordinates with room for a tile; row distances
// are below TMA's 2^40 bytes and keep every 64-bit offset in range.
constexpr int64_t kMaxSize = (int64_t)1 << 30;
constexpr int64_t kMaxLd = (int64_t)1 << 32;

// what a product's epilogue does with the accumulators D[f][t] (f: the output's
// contiguous dimension, t: its row)
enum Kind {
    kForward = 0,     // Y[t][f] = act(D + bias[f]) + add[t][f]; z / z8 keep D + bias
    kGradInput = 1,   // dX[t][f] = D * act'(z[t][f]) + add[t][f]; z comes in 16 bits or as z8; xv keeps act(z)
    kGradWeight = 2,  // dW[t][f] = D + add[t][f] (add: dW itself, of its type)
};

struct Epilogue {
    int m, n;        // f < m, t < n
    int act;
    int out_f32;     // out is FP32 (kGradWeight), else of the operands' type
    float* sums;     // kGradInput: sums of out's columns over parts of its rows, [sum_parts()][m]
    // the product's operands, and how near to +-1/2 a quotient is taken from them (SETTLE); set by gemm() and launch()
    const void *w, *x;
    int64_t ldw, ldx;
    int k;
    float tie;
    bool vec_out, vec_add, vec_z, vec_codes;  // 16-byte (8 for codes) accesses fit; set by gemm()
    void* out;
    int64_t ldo;
    const void* bias;
    const void* add;
    int64_t ldadd;
    void* z;         // 16-bit z: written by kForward, read by kGradInput
    int64_t ldz;
    chpl_ckpt8 z8;   // 8-bit z: written by kForward, read by kGradInput
    void* xv;        // kGradInput: act(z), of the operands' type
    int64_t ldxv;
};

// One operand of a product over c: element (i, c) at p[i * ld + c] when
// k_major, else at p[c * ld + i].  16-bit, base and rows on 16-byte boundaries.
struct Operand {
    const void* p;
    int64_t ld;
    bool k_major;
};

// D[f][t] = sum_{c < k} A(f, c) B(t, c), handed to the epilogue; type BF16 or F16
int gemm(cudaStream_t st, int type, Kind kind, const Operand& a, const Operand& b, int64_t k, const Epilogue& e);

// parts that a product's column sums come in
int64_t sum_parts(int64_t m, int64_t n, int64_t k);

int check_size(const char* who, const char* what, int64_t v);
int check_operand(const char* who, const char* what, const void* p, int64_t ld, int64_t width, int elt);
int check_ckpt(const char* who, const char* what, const chpl_ckpt8& c, int64_t width);
int check_work(const char* who, const void* work, size_t have, size_t need);

// of the products' plans and tensor maps
int num_sms();
int slots(int split, int resident, int sms);
int fit_rows(int n, int bn, int step);
// Estimated time in us (linear_gemm.cu says where it comes from) of `tiles` tiles of
// bn rows, a stage of the contraction taking stage_bytes of each: by clusters of
// `split` CTAs, one or two of them resident on an SM, and by pairs, whose stage is
// the even CTA's with all of the rows.
struct SplitTime {
    double us;
    int resident;
};
SplitTime split_time(int stage_bytes, int bn, int64_t tiles, int split, int kblocks, int sms);
double pair_time(int stage_bytes, int bn, int64_t tiles, int kblocks, int sms);

int read_clear_status(int* st);

}  // namespace linear
}  // namespace chpl
