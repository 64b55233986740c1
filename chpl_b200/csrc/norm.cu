// Norms around a model's blocks (the C entry points chpl_norm_forward and
// chpl_norm_backward): RMS or layer norm of a token's features before a block,
// and the join of a block's output with the residual stream, r = beta x + alpha
// gate * Npost(y), together with the next block's norm h = Npre(r).
//
// Bound: HBM; every row is read and written once.  A row lies in the registers
// of one CTA (of a cluster above 8192 features), eight features a thread, so
// that the statistics' passes over it cost no memory traffic and the gradients'
// sums over the tokens stay in registers, eight a thread, from a CTA's first row
// to its last.  The rows to come are on their way into shared memory meanwhile,
// every thread copying what it will itself read: no barrier waits for a copy.
#include <algorithm>
#include <cmath>

#include "ckpt8.cuh"
#include "linear.h"

namespace chpl {
namespace norm {

using linear::check_operand;
using linear::check_size;

constexpr int kMaxThreads = 1024;
constexpr int kMaxWidth = 2 * 8 * kMaxThreads;  // a cluster of two
constexpr int kMaxStages = 4;
constexpr int kStageBudget = 192 * 1024;        // of shared memory on an SM, for the rows under way

// ----------------------------------------------------------------------------
// shape of a launch
// ----------------------------------------------------------------------------
struct Shape {
    int warps;    // of a row in one CTA
    int groups;   // rows that a CTA holds at once
    int cluster;  // CTAs that share a row
    int stages;   // rows of each group that are under way or in use
    int units;    // clusters launched
    int smem;
};

// A row's warps are a power of two up to four (several rows to a CTA of eight
// warps), then as many as it needs.  64 registers a thread leave 1024 threads on
// an SM.
static Shape shape_for(int64_t tokens, int64_t n, int tensors, int vectors)
{
    Shape s;
    s.cluster = n > 8 * kMaxThreads ? 2 : 1;
    const int need = (int)((n + 256 * s.cluster - 1) / (256 * s.cluster));
    s.warps = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need;
    s.groups = s.warps <= 4 ? 8 / s.warps : 1;
    const int threads = 32 * s.warps * s.groups, resident = kMaxThreads / threads;
    const int fixed = vectors * threads * 16;
    s.stages = std::max(1, std::min(kMaxStages, (kStageBudget / resident - fixed) / std::max(1, tensors * threads * 16)));
    s.smem = fixed + s.stages * tensors * threads * 16;
    const int64_t want = (tokens + s.groups - 1) / s.groups;
    s.units = (int)std::min<int64_t>(want, 148 / s.cluster * resident);
    return s;
}

// ----------------------------------------------------------------------------
// eight features of a thread
// ----------------------------------------------------------------------------
// Features first + (i / E) * stride + i % E of i = 0 .. 7: pieces of E that the
// rows' alignment allows to access at once.
template <int E>
struct Columns {
    int first, stride, n;
    __device__ __forceinline__ int at(int i) const { return first + i / E * stride + i % E; }
    __device__ __forceinline__ bool has(int i) const { return at(i) < n; }
};

// the thread's features of a row (or a vector) into 16 bytes of shared memory,
// zero past the end; asynchronous where pieces are of 4 bytes at least
template <int E>
__device__ __forceinline__ void fetch(uint32_t slot, const void* row, const Columns<E>& c)
{
    const unsigned short* p = static_cast<const unsigned short*>(row);
    if constexpr (E == 1) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c.has(i)) w[i >> 1] |= (uint32_t)p[c.at(i)] << (16 * (i & 1));
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += E) {
            const int left = min(max(c.n - c.at(i), 0), E);
            const void* src = p + (left ? c.at(i) : 0);
            if (E == 8) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot), "l"(src), "r"(2 * left) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(slot + 2 * i), "l"(src), "r"(2 * left) : "memory");
        }
    }
}

template <typename T>
__device__ __forceinline__ void values(uint32_t slot, float (&v)[8])
{
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(slot) : "memory");
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}

template <typename T, int E>
__device__ __forceinline__ void put(void* row, const Columns<E>& c, const float (&v)[8])
{
    T* p = static_cast<T*>(row);
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    const uint32_t* u = &w.x;
#pragma unroll
    for (int i = 0; i < 8; i += E) {
        if (E == 8 && c.has(7)) *reinterpret_cast<uint4*>(p + c.at(0)) = w;
        else if (E == 2 && c.has(i + 1)) *reinterpret_cast<uint32_t*>(p + c.at(i)) = u[i / 2];
        else {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (c.has(i + k)) p[c.at(i + k)] = e[i + k];
        }
    }
}

// ----------------------------------------------------------------------------
// sums over a row
// ----------------------------------------------------------------------------
constexpr int kMaxWarps = kMaxThreads / 32;

// Two sums over the row of a group (of a cluster); every thread of it calls
// with the same count of calls before.  Warps' sums go through shared memory, two
// sets of them in turn: who writes a set again has passed the barrier that all
// readers of its last use reached afterwards.
struct RowSums {
    float2 (*sets)[kMaxWarps];  // [2][warps of the CTA]
    int warps, group, cluster, turn;

    __device__ __forceinline__ float2 operator()(float a, float b)
    {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
            b += __shfl_xor_sync(0xffffffffu, b, d);
        }
        if (warps == 1) return make_float2(a, b);
        float2* set = sets[turn];
        turn ^= 1;
        const int lane = lane_id();
        if (lane == 0) set[warp_id()] = make_float2(a, b);
        if (cluster > 1) cluster_sync();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * warps) : "memory");
        a = b = 0.0f;
        if (lane < warps) {
            if (cluster == 1) {
                const float2 v = set[group * warps + lane];
                a = v.x;
                b = v.y;
            } else {
                for (int r = 0; r < cluster; ++r) {
                    float2 v;
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(map_to_rank(smem_u32(set + lane), (uint32_t)r)) : "memory");
                    a += v.x;
                    b += v.y;
                }
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
            b += __shfl_xor_sync(0xffffffffu, b, d);
        }
        return make_float2(a, b);
    }
};

// where a thread stands
template <int E>
struct Place {
    Columns<E> cols;
    int group;
    int64_t row, step;
    __device__ __forceinline__ Place(const Shape& s, int n)
    {
        const int warp = warp_id(), rank = s.cluster > 1 ? (int)cluster_ctarank() : 0;
        group = warp / s.warps;
        const int thread = (warp - group * s.warps) * 32 + lane_id(), width = 32 * s.warps;
        cols = {rank * width * 8 + thread * E, width * E, n};
        const int64_t unit = blockIdx.x / s.cluster;
        row = unit * s.groups + group;
        step = (int64_t)s.units * s.groups;
    }
};

// The rows under way: copies of the rows to come, a group of cp.async each,
// `stages` of them (an empty group where there is no such row).
struct Ring {
    uint32_t base;  // of the thread
    uint32_t tensor, stage_bytes;
    int stages, at;
    __device__ __forceinline__ Ring(uint32_t smem, int tensors, int nstages)
        : base(smem + threadIdx.x * 16), tensor(blockDim.x * 16), stage_bytes((uint32_t)tensors * blockDim.x * 16), stages(nstages), at(0)
    {
    }
    __device__ __forceinline__ uint32_t slot(int stage, int t) const { return base + stage * stage_bytes + t * tensor; }
    __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // the oldest of `stages` groups has arrived
    __device__ __forceinline__ void wait() const
    {
        switch (stages) {
            case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
            case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
            case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
            default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        }
    }
    __device__ __forceinline__ void next() { at = at + 1 == stages ? 0 : at + 1; }
};

// ----------------------------------------------------------------------------
// forward
// ----------------------------------------------------------------------------
struct Rows {
    const void* p;
    int64_t ld;
    __device__ __forceinline__ const void* row(int64_t t) const { return static_cast<const unsigned short*>(p) + t * ld; }
};
struct RowsTo {
    void* p;
    int64_t ld;
    __device__ __forceinline__ void* row(int64_t t) const { return static_cast<unsigned short*>(p) + t * ld; }
};

struct Forward {
    int64_t tokens;
    int n;
    float scale, residual_scale, post_eps, pre_eps;
    int post, pre;          // kinds
    Rows x, y, gate;        // gate.ld 0: a vector
    const void *post_w, *post_b, *pre_w, *pre_b;
    RowsTo r, h;
    float2 *post_stats, *pre_stats;
};

// slots of the vectors
enum { kPostW, kPostB, kPreW, kPreB, kGate, kVectors };

// the norm of v, in place; (mean, 1 / deviation) to *stats.  Mean first, then the
// squares of what is left: the one pass of squares loses the variance of rows
// whose mean is large.
template <typename T, int E>
__device__ __forceinline__ void normalize(float (&v)[8], const Columns<E>& c, int kind, float eps, float inv_n, uint32_t w, uint32_t b,
                                          bool has_b, RowSums& sums, float2* stats, bool writes)
{
    float mean = 0.0f;
    if (kind == CHPL_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];  // zero past the end
        mean = sums(s, 0.0f).x * inv_n;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] -= mean;
        q += c.has(i) ? v[i] * v[i] : 0.0f;
    }
    const float rstd = rsqrtf(fmaf(sums(q, 0.0f).x, inv_n, eps));
    if (stats && writes) *stats = make_float2(mean, rstd);
    float wv[8], bv[8] = {};
    values<T>(w, wv);
    if (has_b) values<T>(b, bv);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i] * rstd, wv[i], bv[i]);
}

template <typename T, int E, bool JOIN>
__global__ void __launch_bounds__(kMaxThreads) forward_kernel(const __grid_constant__ Forward a, const Shape s)
{
    extern __shared__ uint4 smem[];
    __shared__ float2 sets[2][kMaxWarps];
    const Place<E> at(s, a.n);
    const Columns<E>& c = at.cols;
    const bool matrix = JOIN && a.gate.p && a.gate.ld;
    const int tensors = JOIN ? 2 + matrix : 1;
    const uint32_t mem = smem_u32(smem), vec = mem + threadIdx.x * 16, vec_step = blockDim.x * 16;
    Ring ring(mem + (JOIN ? kVectors : 2) * vec_step, tensors, s.stages);
    RowSums sums = {sets, s.warps, at.group, s.cluster, 0};
    const float inv_n = 1.0f / (float)a.n;
    const uint32_t pre_w = vec + (JOIN ? kPreW : 0) * vec_step, pre_b = vec + (JOIN ? kPreB : 1) * vec_step;
    start_of_inputs();
    if (a.pre) {
        fetch<E>(pre_w, a.pre_w, c);
        if (a.pre_b) fetch<E>(pre_b, a.pre_b, c);
    }
    if (JOIN) {
        if (a.post) {
            fetch<E>(vec + kPostW * vec_step, a.post_w, c);
            if (a.post_b) fetch<E>(vec + kPostB * vec_step, a.post_b, c);
        }
        if (a.gate.p && !matrix) fetch<E>(vec + kGate * vec_step, a.gate.p, c);
    }
    const auto load = [&](int64_t row, int stage) {
        if (row < a.tokens) {
            fetch<E>(ring.slot(stage, 0), a.x.row(row), c);
            if (JOIN) fetch<E>(ring.slot(stage, 1), a.y.row(row), c);
            if (JOIN && matrix) fetch<E>(ring.slot(stage, 2), a.gate.row(row), c);
        }
        Ring::commit();
    };
    for (int i = 0; i < s.stages; ++i) load(at.row + i * at.step, i);
    // writes of a row's statistics: one thread of the row
    const bool writes = c.first == 0;
    for (int64_t row = at.row; row < a.tokens; row += at.step, ring.next()) {
        ring.wait();
        float v[8];
        if (JOIN) {
            values<T>(ring.slot(ring.at, 1), v);
            if (a.post)
                normalize<T, E>(v, c, a.post, a.post_eps, inv_n, vec + kPostW * vec_step, vec + kPostB * vec_step, a.post_b, sums,
                                a.post_stats ? a.post_stats + row : nullptr, writes);
            float u[8];
            if (a.gate.p) {
                values<T>(matrix ? ring.slot(ring.at, 2) : vec + kGate * vec_step, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= u[i];
            }
            values<T>(ring.slot(ring.at, 0), u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c.has(i) ? fmaf(a.scale, v[i], a.residual_scale * u[i]) : 0.0f;
            put<T, E>(a.r.row(row), c, v);
        } else {
            values<T>(ring.slot(ring.at, 0), v);
        }
        load(row + s.stages * at.step, ring.at);
        if (a.pre) {
            normalize<T, E>(v, c, a.pre, a.pre_eps, inv_n, pre_w, pre_b, a.pre_b, sums, a.pre_stats ? a.pre_stats + row : nullptr, writes);
            put<T, E>(a.h.row(row), c, v);
        }
    }
    if (s.cluster > 1) cluster_sync();  // no CTA leaves while another still reads its sums
}

// ----------------------------------------------------------------------------
// backward
// ----------------------------------------------------------------------------
struct Backward {
    int64_t tokens;
    int n;
    float scale, residual_scale;
    int post, pre;
    Rows dr, dh, r, y, gate;  // gate.ld 0: a vector; y.p NULL: no join
    const void *post_w, *post_b, *pre_w;
    const float2 *post_stats, *pre_stats;
    RowsTo dx, dy, dgate;     // dgate of a matrix
    float* part;              // [sum][unit][n] of the sums that `sums` names
    int sums;                 // bit k: sum k
};

// Sums over the tokens, from which the parameters' gradients follow: with Do =
// alpha D (times the gate where it is a matrix), yhat the normed y (or y),
//   0  Do yhat   dw_post = gate * 0,  dgate = w_post * 0 + b_post * 1
//   1  Do        db_post = gate * 1
//   2  dh rhat   dw_pre
//   3  dh        db_pre
constexpr int kSums = 4;

template <typename T, int E, bool JOIN, bool BIAS>
__global__ void __launch_bounds__(kMaxThreads) backward_kernel(const __grid_constant__ Backward a, const Shape s)
{
    extern __shared__ uint4 smem[];
    __shared__ float2 sets[2][kMaxWarps];
    const Place<E> at(s, a.n);
    const Columns<E>& c = at.cols;
    const bool matrix = JOIN && a.gate.p && a.gate.ld, has_y = JOIN && a.y.p;
    const int t_dh = a.dr.p ? 1 : 0, t_r = t_dh + 1, t_y = a.pre ? t_r + 1 : t_dh, t_gate = t_y + has_y, tensors = t_gate + matrix;
    const uint32_t mem = smem_u32(smem), vec = mem + threadIdx.x * 16, vec_step = blockDim.x * 16;
    const uint32_t pre_w = vec, post_w = vec + vec_step, post_b = post_w + vec_step, gate_v = post_b + vec_step;
    Ring ring(mem + (JOIN ? 4 : 1) * vec_step, tensors, s.stages);
    RowSums sums = {sets, s.warps, at.group, s.cluster, 0};
    const float inv_n = 1.0f / (float)a.n;
    start_of_inputs();
    if (a.pre) fetch<E>(pre_w, a.pre_w, c);
    if (JOIN) {
        if (a.post) fetch<E>(post_w, a.post_w, c);
        if (a.post && a.post_b) fetch<E>(post_b, a.post_b, c);
        if (a.gate.p && !matrix) fetch<E>(gate_v, a.gate.p, c);
    }
    const auto load = [&](int64_t row, int stage) {
        if (row < a.tokens) {
            if (a.dr.p) fetch<E>(ring.slot(stage, 0), a.dr.row(row), c);
            if (a.pre) {
                fetch<E>(ring.slot(stage, t_dh), a.dh.row(row), c);
                fetch<E>(ring.slot(stage, t_r), a.r.row(row), c);
            }
            if (has_y) fetch<E>(ring.slot(stage, t_y), a.y.row(row), c);
            if (matrix) fetch<E>(ring.slot(stage, t_gate), a.gate.row(row), c);
        }
        Ring::commit();
    };
    const auto stats_of = [&](int64_t row, float2& pre, float2& post) {
        pre = post = make_float2(0.0f, 1.0f);
        if (row >= a.tokens) return;
        if (a.pre) pre = __ldg(a.pre_stats + row);
        if (JOIN && a.post) post = __ldg(a.post_stats + row);
    };
    float total[BIAS ? kSums : 2][8] = {};  // without biases sums 0 and 2
    constexpr int kHat = BIAS ? 2 : 1;
    float2 pre_next, post_next;
    stats_of(at.row, pre_next, post_next);
    for (int i = 0; i < s.stages; ++i) load(at.row + i * at.step, i);
    for (int64_t row = at.row; row < a.tokens; row += at.step, ring.next()) {
        const float2 pre = pre_next, post = post_next;
        stats_of(row + at.step, pre_next, post_next);
        ring.wait();
        float d[8] = {};
        if (a.pre) {
            float g[8], hat[8], w[8];
            values<T>(ring.slot(ring.at, t_dh), g);
            values<T>(ring.slot(ring.at, t_r), hat);
            values<T>(pre_w, w);
            float sg = 0.0f, sgh = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                hat[i] = c.has(i) ? (hat[i] - pre.x) * pre.y : 0.0f;
                total[kHat][i] = fmaf(g[i], hat[i], total[kHat][i]);
                if constexpr (BIAS) total[3][i] += g[i];
                g[i] *= w[i];
                sg += g[i];
                sgh = fmaf(g[i], hat[i], sgh);
            }
            const float2 m = sums(sg, sgh);
            const float mg = a.pre == CHPL_NORM_LAYER ? m.x * inv_n : 0.0f, mgh = m.y * inv_n;
            if (a.dr.p) values<T>(ring.slot(ring.at, 0), d);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = fmaf(pre.y, fmaf(-hat[i], mgh, g[i] - mg), d[i]);
        } else {
            values<T>(ring.slot(ring.at, 0), d);
        }
        if (a.dx.p) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = JOIN ? a.residual_scale * d[i] : d[i];
            put<T, E>(a.dx.row(row), c, o);
        }
        if (JOIN) {
            float y[8] = {}, w[8], u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = c.has(i) ? a.scale * d[i] : 0.0f;
            if (has_y) values<T>(ring.slot(ring.at, t_y), y);
            if (a.post) {
                values<T>(post_w, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = c.has(i) ? (y[i] - post.x) * post.y : 0.0f;
            }
            if (matrix) {
                values<T>(ring.slot(ring.at, t_gate), u);
                if (a.dgate.p) {
                    float o[8], b[8] = {};
                    if (a.post && a.post_b) values<T>(post_b, b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = d[i] * (a.post ? fmaf(y[i], w[i], b[i]) : y[i]);
                    put<T, E>(a.dgate.row(row), c, o);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= u[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                total[0][i] = fmaf(d[i], y[i], total[0][i]);
                if constexpr (BIAS) total[1][i] += d[i];
            }
            if (a.gate.p && !matrix) {
                values<T>(gate_v, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= u[i];
            }
            load(row + s.stages * at.step, ring.at);
            if (a.post) {
                float sg = 0.0f, sgh = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d[i] *= w[i];
                    sg += d[i];
                    sgh = fmaf(d[i], y[i], sgh);
                }
                const float2 m = sums(sg, sgh);
                const float mg = a.post == CHPL_NORM_LAYER ? m.x * inv_n : 0.0f, mgh = m.y * inv_n;
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = post.y * fmaf(-y[i], mgh, d[i] - mg);
            }
            if (a.dy.p) put<T, E>(a.dy.row(row), c, d);
        } else {
            load(row + s.stages * at.step, ring.at);
        }
    }
    // a CTA's sums: those of its groups, joined in shared memory in order
    if (a.part) {
        float* turn = reinterpret_cast<float*>(smem);  // [groups][8][threads of a group]
        const int width = 32 * s.warps, thread = threadIdx.x - at.group * width;
        const int64_t unit = blockIdx.x / s.cluster;
        asm volatile("cp.async.wait_all;" ::: "memory");
        int slot = 0;
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            if (!(a.sums >> k & 1)) continue;
            const int have = BIAS ? k : k / 2;
            if (s.groups > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) turn[(at.group * 8 + i) * width + thread] = total[have][i];
                __syncthreads();
            }
            if (at.group == 0) {
                float* out = a.part + ((int64_t)slot * s.units + unit) * a.n;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v = total[have][i];
                    for (int g = 1; g < s.groups; ++g) v += turn[(g * 8 + i) * width + thread];
                    if (c.has(i)) out[c.at(i)] = v;
                }
            }
            ++slot;
        }
    }
    if (s.cluster > 1) cluster_sync();
}

// The parameters' gradients from the units' sums.  A block takes 32 features, its
// warps equal runs of the units, joined in order; bound by the loads' latency.
struct Parameters {
    const float* part;
    int units, n, sums;
    int f32, accumulate, matrix;
    const void *post_w, *post_b, *gate;  // as they were used
    void *dpost_w, *dpost_b, *dgate, *dpre_w, *dpre_b;
};

constexpr int kJoinWarps = 16;

template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) parameters_kernel(const __grid_constant__ Parameters a)
{
    __shared__ float turn[kSums][kJoinWarps][32];
    const int lane = lane_id(), warp = warp_id(), j = blockIdx.x * 32 + lane;
    const int first = (int)((int64_t)a.units * warp / kJoinWarps), last = (int)((int64_t)a.units * (warp + 1) / kJoinWarps);
    start_of_inputs();
    float sum[kSums] = {};
    int slot = 0;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        if (!(a.sums >> k & 1)) continue;
        const float* p = a.part + (int64_t)slot++ * a.units * a.n + j;
        if (j < a.n) {
#pragma unroll 8
            for (int u = first; u < last; ++u) sum[k] += p[(int64_t)u * a.n];
        }
        turn[k][warp][lane] = sum[k];
    }
    __syncthreads();
    if (warp > 0 || j >= a.n) return;
#pragma unroll
    for (int k = 0; k < kSums; ++k)
        if (a.sums >> k & 1)
            for (int w = 1; w < kJoinWarps; ++w) sum[k] += turn[k][w][lane];
    const auto of = [&](const void* v, float other) { return v ? to_f32(static_cast<const T*>(v)[j]) : other; };
    const auto store = [&](void* out, float v) {
        if (!out) return;
        if (a.f32) {
            float* o = static_cast<float*>(out) + j;
            *o = a.accumulate ? *o + v : v;
        } else {
            T* o = static_cast<T*>(out) + j;
            *o = from_f32<T>(a.accumulate ? to_f32(*o) + v : v);
        }
    };
    const float gate = a.matrix ? 1.0f : of(a.gate, 1.0f);  // a matrix is in the sums
    store(a.dpost_w, gate * sum[0]);
    store(a.dpost_b, gate * sum[1]);
    store(a.dgate, fmaf(of(a.post_w, 1.0f), sum[0], a.post_b ? of(a.post_b, 0.0f) * sum[1] : 0.0f));
    store(a.dpre_w, sum[2]);
    store(a.dpre_b, sum[3]);
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static int check_norm(const char* who, const char* what, const chpl_norm& v, int64_t n, bool pointers)
{
    if (v.kind < CHPL_NORM_NONE || v.kind > CHPL_NORM_LAYER) { set_error("%s: unknown kind %d of the norm %s", who, v.kind, what); return CHPL_ERR_INVALID; }
    if (v.kind == CHPL_NORM_NONE) return CHPL_OK;
    if (!(v.eps >= 0.0f) || !(v.eps < INFINITY)) { set_error("%s: eps of the norm %s is %g", who, what, v.eps); return CHPL_ERR_INVALID; }
    if (!pointers || n == 0) return CHPL_OK;
    CHPL_TRY(check_operand(who, "a norm's weight", v.weight, n, n, 2));
    if (v.bias) CHPL_TRY(check_operand(who, "a norm's bias", v.bias, n, n, 2));
    return CHPL_OK;
}

static int check_common(const char* who, int type, int64_t tokens, int64_t n, float scale, float residual_scale)
{
    if (type != CHPL_TYPE_BF16 && type != CHPL_TYPE_F16) { set_error("%s: type %d is not BF16 or F16", who, type); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_size(who, "tokens", tokens));
    CHPL_TRY(check_size(who, "n", n));
    if (n > kMaxWidth) { set_error("%s: n = %lld exceeds %d", who, (long long)n, kMaxWidth); return CHPL_ERR_UNSUPPORTED; }
    if (!std::isfinite(scale) || !std::isfinite(residual_scale)) { set_error("%s: a scale is not finite", who); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

static int check_stats(const char* who, const char* what, const void* p, bool needed)
{
    if (needed && !p) { set_error("%s: %s are NULL", who, what); return CHPL_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(p) % 8) { set_error("%s: %s are not 8-byte aligned", who, what); return CHPL_ERR_INVALID; }
    return CHPL_OK;
}

// features that all rows can be accessed by at once: 8, 2 or 1
struct Pieces {
    int e = 8;
    void add(const void* p, int64_t ld, int64_t tokens)
    {
        if (!p) return;
        const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (tokens > 1 ? (uintptr_t)(ld * 2) : 0);
        e = std::min(e, a % 16 == 0 ? 8 : a % 4 == 0 ? 2 : 1);
    }
};

static int check(const char* who, const chpl_norm_fwd* a)
{
    if (!a) { set_error("%s: arguments are NULL", who); return CHPL_ERR_INVALID; }
    const bool any = a->tokens > 0 && a->n > 0;
    CHPL_TRY(check_common(who, a->type, a->tokens, a->n, a->scale, a->residual_scale));
    CHPL_TRY(check_norm(who, "of y", a->post, a->n, any));
    CHPL_TRY(check_norm(who, "of the sum", a->pre, a->n, any));
    if (a->pre.kind == CHPL_NORM_NONE && !a->join) { set_error("%s: neither a norm nor a join", who); return CHPL_ERR_INVALID; }
    if (!a->join && a->post.kind != CHPL_NORM_NONE) { set_error("%s: a norm of y without a join", who); return CHPL_ERR_INVALID; }
    if (!any) return CHPL_OK;
    CHPL_TRY(check_operand(who, "x", a->x, a->ldx, a->n, 2));
    if (a->join) {
        CHPL_TRY(check_operand(who, "y", a->y, a->ldy, a->n, 2));
        CHPL_TRY(check_operand(who, "r", a->r, a->ldr, a->n, 2));
        if (a->gate) CHPL_TRY(check_operand(who, "gate", a->gate, a->ldgate ? a->ldgate : a->n, a->n, 2));
        if ((a->r == a->x && a->ldr != a->ldx) || (a->r == a->y && a->ldr != a->ldy)) { set_error("%s: r is an input with another row distance", who); return CHPL_ERR_INVALID; }
        CHPL_TRY(check_stats(who, "statistics of y", a->post_stats, false));
    }
    if (a->pre.kind != CHPL_NORM_NONE) {
        CHPL_TRY(check_operand(who, "h", a->h, a->ldh, a->n, 2));
        if ((a->h == a->x && a->ldh != a->ldx) || (a->join && a->h == a->y && a->ldh != a->ldy)) { set_error("%s: h is an input with another row distance", who); return CHPL_ERR_INVALID; }
        if (a->join && a->h == a->r) { set_error("%s: h and r are the same", who); return CHPL_ERR_INVALID; }
        CHPL_TRY(check_stats(who, "statistics of the sum", a->pre_stats, false));
    }
    return CHPL_OK;
}

template <auto KERNEL, typename A>
static int launch(cudaStream_t st, const A& a, const Shape& s)
{
    static std::atomic<uint64_t> ready{0};
    CHPL_TRY(allow_smem(KERNEL, kStageBudget, ready));
    return launch_kernel(KERNEL, (int64_t)s.units * s.cluster, 32 * s.warps * s.groups, s.smem, s.cluster, st, a, s);
}

template <typename T, bool JOIN>
static int forward(cudaStream_t st, int pieces, const Forward& f, const Shape& s)
{
    if (pieces == 8) return launch<forward_kernel<T, 8, JOIN>>(st, f, s);
    if (pieces == 2) return launch<forward_kernel<T, 2, JOIN>>(st, f, s);
    return launch<forward_kernel<T, 1, JOIN>>(st, f, s);
}

template <typename T>
static int forward(cudaStream_t st, const chpl_norm_fwd& a)
{
    Forward f = {};
    f.tokens = a.tokens;
    f.n = (int)a.n;
    f.scale = a.scale;
    f.residual_scale = a.residual_scale;
    f.pre = a.pre.kind;
    f.pre_eps = a.pre.eps;
    f.x = {a.x, a.ldx};
    Pieces p;
    p.add(a.x, a.ldx, a.tokens);
    if (a.join) {
        f.post = a.post.kind;
        f.post_eps = a.post.eps;
        f.y = {a.y, a.ldy};
        f.gate = {a.gate, a.ldgate};
        f.r = {a.r, a.ldr};
        p.add(a.y, a.ldy, a.tokens);
        p.add(a.r, a.ldr, a.tokens);
        p.add(a.gate, a.ldgate, a.tokens);
        if (f.post) {
            f.post_w = a.post.weight;
            f.post_b = a.post.bias;
            f.post_stats = reinterpret_cast<float2*>(a.post_stats);
            p.add(f.post_w, 0, 1);
            p.add(f.post_b, 0, 1);
        }
    }
    if (f.pre) {
        f.pre_w = a.pre.weight;
        f.pre_b = a.pre.bias;
        f.h = {a.h, a.ldh};
        f.pre_stats = reinterpret_cast<float2*>(a.pre_stats);
        p.add(f.pre_w, 0, 1);
        p.add(f.pre_b, 0, 1);
        p.add(a.h, a.ldh, a.tokens);
    }
    const Shape s = shape_for(a.tokens, a.n, a.join ? 2 + (a.gate && a.ldgate) : 1, a.join ? kVectors : 2);
    return a.join ? forward<T, true>(st, p.e, f, s) : forward<T, false>(st, p.e, f, s);
}

// what a backward call forms
struct BackwardPlan {
    Shape shape;
    int sums;        // bits
    size_t bytes;
};

static BackwardPlan plan(const chpl_norm_bwd& a)
{
    BackwardPlan p;
    const bool vector_gate = a.dgate && a.gate && a.ldgate == 0;
    p.sums = 0;
    if (a.join && ((a.post.kind && a.dpost_weight) || vector_gate)) p.sums |= 1;
    if (a.join && a.post.kind && (a.dpost_bias || (vector_gate && a.post.bias))) p.sums |= 2;
    if (a.pre.kind && a.dpre_weight) p.sums |= 4;
    if (a.pre.kind && a.dpre_bias) p.sums |= 8;
    int tensors = (a.dr ? 1 : 0) + (a.pre.kind ? 2 : 0);
    if (a.join) tensors += (a.post.kind || a.gate ? 1 : 0) + (a.gate && a.ldgate ? 1 : 0);
    p.shape = shape_for(a.tokens, a.n, tensors, a.join ? 4 : 1);
    // the groups' sums are joined where the rows under way were
    p.shape.smem = std::max(p.shape.smem, p.shape.groups > 1 ? 32 * p.shape.warps * p.shape.groups * 8 * 4 : 0);
    int count = 0;
    for (int k = 0; k < kSums; ++k) count += p.sums >> k & 1;
    p.bytes = round_up((size_t)count * p.shape.units * a.n * 4, 256);
    return p;
}

static int check(const char* who, const chpl_norm_bwd* a, bool pointers)
{
    if (!a) { set_error("%s: arguments are NULL", who); return CHPL_ERR_INVALID; }
    const bool any = pointers && a->tokens > 0 && a->n > 0;
    CHPL_TRY(check_common(who, a->type, a->tokens, a->n, a->scale, a->residual_scale));
    if (a->grad_type != a->type && a->grad_type != CHPL_TYPE_F32) { set_error("%s: grad_type %d is neither the operands' type nor F32", who, a->grad_type); return CHPL_ERR_INVALID; }
    CHPL_TRY(check_norm(who, "of y", a->post, a->n, any));
    CHPL_TRY(check_norm(who, "of the sum", a->pre, a->n, any));
    if (a->pre.kind == CHPL_NORM_NONE && !a->join) { set_error("%s: neither a norm nor a join", who); return CHPL_ERR_INVALID; }
    if (!a->join && a->post.kind != CHPL_NORM_NONE) { set_error("%s: a norm of y without a join", who); return CHPL_ERR_INVALID; }
    if ((a->dpre_weight || a->dpre_bias) && a->pre.kind == CHPL_NORM_NONE) { set_error("%s: gradients of a norm of the sum that there is not", who); return CHPL_ERR_INVALID; }
    if ((a->dpost_weight || a->dpost_bias) && (!a->join || a->post.kind == CHPL_NORM_NONE)) { set_error("%s: gradients of a norm of y that there is not", who); return CHPL_ERR_INVALID; }
    if (a->dgate && (!a->join || !a->gate)) { set_error("%s: dgate without a gate", who); return CHPL_ERR_INVALID; }
    if (!a->join && a->dy) { set_error("%s: dy without a join", who); return CHPL_ERR_INVALID; }
    if (!pointers) return CHPL_OK;
    const int ge = a->grad_type == CHPL_TYPE_F32 ? 4 : 2;
    if (a->n > 0) {
        if (a->dpre_weight) CHPL_TRY(check_operand(who, "dweight of the sum's norm", a->dpre_weight, a->n, a->n, ge));
        if (a->dpre_bias) CHPL_TRY(check_operand(who, "dbias of the sum's norm", a->dpre_bias, a->n, a->n, ge));
        if (a->dpost_weight) CHPL_TRY(check_operand(who, "dweight of y's norm", a->dpost_weight, a->n, a->n, ge));
        if (a->dpost_bias) CHPL_TRY(check_operand(who, "dbias of y's norm", a->dpost_bias, a->n, a->n, ge));
        if (a->dgate && !a->ldgate) CHPL_TRY(check_operand(who, "dgate", a->dgate, a->n, a->n, ge));
        // without tokens the parameters' gradients still follow from these
        if (a->join && a->gate && !a->ldgate) CHPL_TRY(check_operand(who, "gate", a->gate, a->n, a->n, 2));
    }
    if (!any) return CHPL_OK;
    if (a->dr) CHPL_TRY(check_operand(who, "dr", a->dr, a->lddr, a->n, 2));
    if (a->pre.kind != CHPL_NORM_NONE) {
        CHPL_TRY(check_operand(who, "dh", a->dh, a->lddh, a->n, 2));
        CHPL_TRY(check_operand(who, "r", a->r, a->ldr, a->n, 2));
        CHPL_TRY(check_stats(who, "statistics of the sum", a->pre_stats, true));
    } else if (!a->dr) {
        set_error("%s: neither dr nor dh", who);
        return CHPL_ERR_INVALID;
    }
    if (a->dx) CHPL_TRY(check_operand(who, "dx", a->dx, a->lddx, a->n, 2));
    if (a->dx && ((a->dx == a->dr && a->lddx != a->lddr) || (a->pre.kind && a->dx == a->dh && a->lddx != a->lddh))) { set_error("%s: dx is an input with another row distance", who); return CHPL_ERR_INVALID; }
    if (a->join) {
        if (a->gate && a->ldgate) CHPL_TRY(check_operand(who, "gate", a->gate, a->ldgate, a->n, 2));
        if (a->post.kind || a->gate) CHPL_TRY(check_operand(who, "y", a->y, a->ldy, a->n, 2));
        if (a->post.kind) CHPL_TRY(check_stats(who, "statistics of y", a->post_stats, true));
        if (a->dy) CHPL_TRY(check_operand(who, "dy", a->dy, a->lddy, a->n, 2));
        if (a->dgate && a->ldgate) CHPL_TRY(check_operand(who, "dgate", a->dgate, a->lddgate, a->n, 2));
    }
    return CHPL_OK;
}

template <typename T, bool JOIN, bool BIAS>
static int backward(cudaStream_t st, int pieces, const Backward& b, const Shape& s)
{
    if (pieces == 8) return launch<backward_kernel<T, 8, JOIN, BIAS>>(st, b, s);
    if (pieces == 2) return launch<backward_kernel<T, 2, JOIN, BIAS>>(st, b, s);
    return launch<backward_kernel<T, 1, JOIN, BIAS>>(st, b, s);
}

template <typename T>
static int backward(cudaStream_t st, const chpl_norm_bwd& a, void* work)
{
    const BackwardPlan plan_ = plan(a);
    const bool matrix = a.join && a.gate && a.ldgate;
    if (a.tokens > 0) {
        Backward b = {};
        b.tokens = a.tokens;
        b.n = (int)a.n;
        b.scale = a.scale;
        b.residual_scale = a.residual_scale;
        b.sums = plan_.sums;
        b.part = plan_.sums ? static_cast<float*>(work) : nullptr;
        b.dr = {a.dr, a.lddr};
        b.dx = {a.dx, a.lddx};
        Pieces p;
        p.add(a.dr, a.lddr, a.tokens);
        p.add(a.dx, a.lddx, a.tokens);
        if (a.pre.kind) {
            b.pre = a.pre.kind;
            b.dh = {a.dh, a.lddh};
            b.r = {a.r, a.ldr};
            b.pre_w = a.pre.weight;
            b.pre_stats = reinterpret_cast<const float2*>(a.pre_stats);
            p.add(a.dh, a.lddh, a.tokens);
            p.add(a.r, a.ldr, a.tokens);
            p.add(b.pre_w, 0, 1);
        }
        if (a.join) {
            if (a.post.kind || a.gate) b.y = {a.y, a.ldy};
            b.gate = {a.gate, a.ldgate};
            b.dy = {a.dy, a.lddy};
            if (matrix) b.dgate = {a.dgate, a.lddgate};
            p.add(b.y.p, b.y.ld, a.tokens);
            p.add(a.gate, a.ldgate, a.tokens);
            p.add(a.dy, a.lddy, a.tokens);
            p.add(b.dgate.p, b.dgate.ld, a.tokens);
            if (a.post.kind) {
                b.post = a.post.kind;
                b.post_w = a.post.weight;
                b.post_b = a.post.bias;
                b.post_stats = reinterpret_cast<const float2*>(a.post_stats);
                p.add(b.post_w, 0, 1);
                p.add(b.post_b, 0, 1);
            }
        }
        const bool bias = (plan_.sums & 10) != 0;
        if (!a.join) CHPL_TRY((backward<T, false, true>(st, p.e, b, plan_.shape)));
        else if (bias) CHPL_TRY((backward<T, true, true>(st, p.e, b, plan_.shape)));
        else CHPL_TRY((backward<T, true, false>(st, p.e, b, plan_.shape)));
    }
    if (!plan_.sums || (a.tokens == 0 && a.accumulate)) return CHPL_OK;
    Parameters q = {};
    q.part = static_cast<const float*>(work);
    q.units = a.tokens > 0 ? plan_.shape.units : 0;
    q.n = (int)a.n;
    q.sums = plan_.sums;
    q.f32 = a.grad_type == CHPL_TYPE_F32;
    q.accumulate = a.accumulate;
    q.matrix = matrix;
    if (a.join) {
        q.gate = a.gate;
        if (!matrix) q.dgate = a.dgate;
        if (a.post.kind) {
            q.post_w = a.post.weight;
            q.post_b = a.post.bias;
            q.dpost_w = a.dpost_weight;
            q.dpost_b = a.dpost_bias;
        }
    }
    if (a.pre.kind) {
        q.dpre_w = a.dpre_weight;
        q.dpre_b = a.dpre_bias;
    }
    return launch_kernel(parameters_kernel<T>, (a.n + 31) / 32, 32 * kJoinWarps, 0, 1, st, q);
}

}  // namespace norm
}  // namespace chpl

extern "C" int chpl_norm_forward(void* stream, const chpl_norm_fwd* a)
{
    using namespace chpl::norm;
    CHPL_TRY(check("norm_forward", a));
    if (a->tokens == 0 || a->n == 0) return CHPL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->type == CHPL_TYPE_BF16 ? forward<__nv_bfloat16>(st, *a) : forward<__half>(st, *a);
}

extern "C" int chpl_norm_backward_worksize(const chpl_norm_bwd* a, size_t* work_bytes)
{
    using namespace chpl::norm;
    CHPL_TRY(check("norm_backward_worksize", a, false));
    if (!work_bytes) { chpl::set_error("norm_backward_worksize: work_bytes is NULL"); return CHPL_ERR_INVALID; }
    *work_bytes = a->tokens == 0 || a->n == 0 ? 0 : plan(*a).bytes;
    return CHPL_OK;
}

extern "C" int chpl_norm_backward(void* stream, const chpl_norm_bwd* a, void* work, size_t work_bytes)
{
    using namespace chpl::norm;
    CHPL_TRY(check("norm_backward", a, true));
    if (a->n == 0) return CHPL_OK;
    const size_t need = a->tokens == 0 ? 0 : plan(*a).bytes;
    CHPL_TRY(chpl::linear::check_work("norm_backward", work, work_bytes, need));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->type == CHPL_TYPE_BF16 ? backward<__nv_bfloat16>(st, *a, work) : backward<__half>(st, *a, work);
}
