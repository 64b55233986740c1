// Norms around a model's blocks (the C entry points chpl_norm_forward and
// chpl_norm_backward): RMS or layer norm of a token's features before a block,
// and the join of a block's output with the residual stream, r = beta x + alpha
// gate * Npost(y), together with the next block's norm h = Npre(r).
//
// Bound: HBM; every row is read and written once.  A row lies in the registers
// of one CTA (a wide one of a cluster), sixteen features a thread, so that the
// statistics' passes over it cost no memory traffic and the gradients' sums over
// the tokens stay in registers from a CTA's first row to its last.  Sixteen,
// because what a row costs a thread beside its features (sums over the row,
// addresses, waits) bounds the kernels with eight: join of 8192 x 4096 68 -> 59 us,
// its gradients 136 -> 101 by that step.  The rows to come are on their way into
// shared memory meanwhile, every warp copying what it will itself read: no barrier
// waits for a copy.
//
// Measured (BF16, from launch to launch): 8192 x 4096 with two RMS norms and a
// vector gate 47.5 us (5.7 TB/s), its gradients 71.5 (5.6); layer norm's gradients
// with a skip's 51.7 (5.2, the launch for the parameters in it); a copy by torch 6.05
// TB/s.  What is left is the latency of the sums over a row, and rows below 512
// features, of which a warp takes as long as for 512.
#include <algorithm>
#include <cmath>

#include "linear_epilogue.cuh"

namespace chpl {
namespace norm {

using linear::check_operand;
using linear::check_size;

constexpr int kHalves = 2;                          // eights of a thread's features, 256 apart
constexpr int kWarpWidth = 256 * kHalves;
constexpr int kForwardThreads = 1024;               // of a CTA, one to an SM: 64 registers each
constexpr int kBackwardThreads = 512;               // 128
constexpr int kMaxWarps = kForwardThreads / 32;
constexpr int kMaxWidth = kForwardThreads * 8 * kHalves;
constexpr int kMaxCluster = 4;
constexpr int kClusterGroups = 4;                   // of a CTA in a cluster
constexpr int kMaxStages = 2;                       // four: gradients of 8192 x 4096 53.8 us, not 51.7
constexpr int kVectorBytes = 1024 * kHalves;        // of a warp's features as FP32
constexpr int kSms = 148;                           // what launches and the workspace are laid out for
constexpr int kSmem = 227 * 1024;                   // of an SM
constexpr int kSmemApart = 2304;                    // of which a CTA takes, beside what it asks for, in whole lines

// ----------------------------------------------------------------------------
// shape of a launch
// ----------------------------------------------------------------------------
struct Shape {
    int warps;    // of a row in one CTA
    int groups;   // rows that a CTA holds at once
    int cluster;  // CTAs that share a row
    int stages;   // rows of each group that are under way or in use
    int units;    // clusters launched
    int piece;    // shared memory of a warp's features
    int turn;     // offset of the memory that unaligned rows are turned about in
    int smem;
};

// One CTA to an SM, of as many groups of warps as its registers hold, each with a
// row of its own: they share the weights in shared memory, and one computes while
// another waits for its row's sums.  A cluster of two or four CTAs shares a row
// where that keeps clearly more of the GPU's threads at work (or where a row and
// the weights do not fit into one CTA's shared memory): gradients of a join with two
// norms, 13107 x 5120, take 14 % less in clusters of two (three groups of five warps)
// than alone (one of ten), 8192 x 8192 the same, 5461 x 12288 7 % more in clusters of
// four than of two.
static Shape shape_for(int64_t tokens, int64_t n, int tensors, int vectors, bool inputs_aligned, bool outputs_aligned, int threads)
{
    constexpr int kNamed = 15;  // named barriers, one to a group of several warps
    Shape s, best = {};
    double most = 0.0;
    int row = 0, fixed = 0, turn = 0;
    const auto sizes = [&] {
        row = std::max(1, tensors) * s.warps * s.piece;
        fixed = vectors * s.warps * kVectorBytes;
        turn = outputs_aligned ? 0 : s.warps * 512;
    };
    s.piece = inputs_aligned ? 1024 : 1056;
    for (s.cluster = 1; s.cluster <= kMaxCluster; s.cluster *= 2) {
        s.warps = (int)((n + kWarpWidth * s.cluster - 1) / (kWarpWidth * s.cluster));
        s.groups = threads / 32 / s.warps;
        if (s.cluster > 1 || s.warps > 1) s.groups = std::min(s.groups, s.cluster > 1 ? kClusterGroups : kNamed);
        sizes();
        if (s.groups == 0 || fixed + turn + row > kSmem - kSmemApart) continue;
        const double work = (double)s.groups * n / s.cluster * linear::slots(s.cluster, 1, kSms);
        if (work <= 1.1 * most) continue;
        most = work;
        best = s;
    }
    s = best;
    sizes();
    // no more groups than hold all rows at once, over the units that run at once: 74
    // clusters of two, 33 of four (join's gradients of 148 x 5120 11.0 us, of 148 x 9216
    // 13.8; 14.2 and 20.4 with the rows dealt out as if to 148 units, one after another)
    const int places = linear::slots(s.cluster, 1, kSms) / s.cluster;
    s.groups = (int)std::max<int64_t>(1, std::min<int64_t>(s.groups, (tokens + places - 1) / places));
    // fewer groups rather than one row under way
    const auto stages = [&] { return (kSmem - kSmemApart - fixed - s.groups * turn) / (s.groups * row); };
    while (s.groups > 1 && stages() < 2) --s.groups;
    s.stages = std::max(1, std::min(kMaxStages, stages()));
    s.turn = fixed + s.groups * s.stages * row;
    s.smem = s.turn + s.groups * turn;
    const int64_t want = (tokens + s.groups - 1) / s.groups;
    s.units = (int)std::min<int64_t>(want, places);
    return s;
}

// ----------------------------------------------------------------------------
// a thread's features: eight consecutive ones in each half of its warp's
// ----------------------------------------------------------------------------
constexpr int kTwos = 4 * kHalves;
struct Some {
    Two v[kTwos];
};

__device__ __forceinline__ Some zeros()
{
    Some r;
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = both(0.0f);
    return r;
}
__device__ __forceinline__ Some operator*(const Some& a, const Some& b)
{
    Some r;
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = a.v[i] * b.v[i];
    return r;
}
__device__ __forceinline__ Some operator+(const Some& a, const Some& b)
{
    Some r;
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = a.v[i] + b.v[i];
    return r;
}
__device__ __forceinline__ Some operator*(const Some& a, float b)
{
    Some r;
    const Two c = both(b);
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = a.v[i] * c;
    return r;
}
__device__ __forceinline__ Some operator+(const Some& a, float b)
{
    Some r;
    const Two c = both(b);
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = a.v[i] + c;
    return r;
}
__device__ __forceinline__ Some fma_of(const Some& a, const Some& b, const Some& c)
{
    Some r;
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = fma2(a.v[i], b.v[i], c.v[i]);
    return r;
}
__device__ __forceinline__ Some fma_of(const Some& a, float b, const Some& c)
{
    Some r;
    const Two m = both(b);
#pragma unroll
    for (int i = 0; i < kTwos; ++i) r.v[i] = fma2(a.v[i], m, c.v[i]);
    return r;
}
__device__ __forceinline__ float total_of(const Some& a)
{
    Two even = a.v[0], odd = a.v[1];
#pragma unroll
    for (int i = 2; i < kTwos; i += 2) {
        even = even + a.v[i];
        odd = odd + a.v[i + 1];
    }
    const float2 t = apart(even + odd);
    return t.x + t.y;
}
__device__ __forceinline__ float dot(const Some& a, const Some& b)
{
    Two even = a.v[0] * b.v[0], odd = a.v[1] * b.v[1];
#pragma unroll
    for (int i = 2; i < kTwos; i += 2) {
        even = fma2(a.v[i], b.v[i], even);
        odd = fma2(a.v[i + 1], b.v[i + 1], odd);
    }
    const float2 t = apart(even + odd);
    return t.x + t.y;
}

// where a thread stands: its features first + 256 h + 0 .. 7, of which left - 256 h
// exist (all eight, some or none)
struct Place {
    int first, left;
    int group;
    uint32_t row, step;  // rows and steps past the last row stay far below 2^32
    __device__ __forceinline__ Place(const Shape& s, int n)
    {
        const int warp = warp_id(), rank = s.cluster > 1 ? (int)cluster_ctarank() : 0;
        group = warp / s.warps;
        first = (rank * s.warps + warp - group * s.warps) * kWarpWidth + lane_id() * 8;
        left = n - first;
        row = blockIdx.x / (uint32_t)s.cluster * s.groups + group;
        step = (uint32_t)(s.units * s.groups);
    }
    __device__ __forceinline__ int have(int h) const { return min(8, max(0, left - 256 * h)); }
    __device__ __forceinline__ bool whole() const { return left >= 256 * (kHalves - 1) + 8; }
};

// zero past the row's end
__device__ __forceinline__ void clear_tail(Some& a, const Place& at)
{
#pragma unroll
    for (int i = 0; i < kTwos; ++i) {
        const float2 t = apart(a.v[i]);
        const int left = at.left - 256 * (i / 4) - 2 * (i % 4);
        a.v[i] = two(left > 0 ? t.x : 0.0f, left > 1 ? t.y : 0.0f);
    }
}

template <typename T>
__device__ __forceinline__ void expand(const uint32_t (&w)[4], int h, Some& r)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = linear::unpack2<T>(w[i]);
        r.v[4 * h + i] = two(f.x, f.y);
    }
}

// features of a warp's 1024 bytes of shared memory in order; at: the lane's first
// (one address register for all of an operand's accesses, here and below: join of
// 16384 x 4096 99.5 -> 97.9 us)
static_assert(kHalves == 2, "the accesses below");
template <typename T>
__device__ __forceinline__ Some packed_at(uint32_t at)
{
    Some r;
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    expand<T>(w, 0, r);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + 512];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    expand<T>(w, 1, r);
    return r;
}

// The thread's features of a vector as they are in memory, zero past the end; all
// ones where there is no vector.
template <typename T>
struct Raw {
    uint32_t w[kHalves][4];
};
template <typename T>
__device__ __forceinline__ Raw<T> raw_vector(const void* v, bool there, const Place& at)
{
    constexpr uint32_t one = std::is_same<T, __half>::value ? 0x3C00u : 0x3F80u;
    Raw<T> r;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        const unsigned short* p = static_cast<const unsigned short*>(v) + at.first + 256 * h;
        const int have = at.have(h);
        if (there && have == 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
            r.w[h][0] = q.x;
            r.w[h][1] = q.y;
            r.w[h][2] = q.z;
            r.w[h][3] = q.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t lo = i < have ? (there ? __ldg(p + i) : one) : 0u, hi = i + 1 < have ? (there ? __ldg(p + i + 1) : one) : 0u;
                r.w[h][i / 2] = lo | hi << 16;
            }
        }
    }
    return r;
}

// A vector, times another (exact in FP32) and a factor, as FP32 in the warp's 2048
// bytes of shared memory, the lane's own: a row then costs neither conversions nor
// the products.  (All of a kernel's vectors are read before the first is put: one
// latency, not one for each, which a single row waits for.)
template <typename T>
__device__ __forceinline__ void put_vector(uint32_t at, const Raw<T>& u, const Raw<T>& v, float factor)
{
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float2 a = linear::unpack2<T>(u.w[h][i]), b = linear::unpack2<T>(u.w[h][i + 1]), c = linear::unpack2<T>(v.w[h][i]),
                         d = linear::unpack2<T>(v.w[h][i + 1]);
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + h * 1024 + i * 256), "f"(a.x * c.x * factor),
                         "f"(a.y * c.y * factor), "f"(b.x * d.x * factor), "f"(b.y * d.y * factor)
                         : "memory");
        }
}
__device__ __forceinline__ Some vector_at(uint32_t at)
{
    Some r;
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(r.v[0].v), "=l"(r.v[1].v) : "r"(at) : "memory");
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2 + 512];" : "=l"(r.v[2].v), "=l"(r.v[3].v) : "r"(at) : "memory");
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2 + 1024];" : "=l"(r.v[4].v), "=l"(r.v[5].v) : "r"(at) : "memory");
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2 + 1536];" : "=l"(r.v[6].v), "=l"(r.v[7].v) : "r"(at) : "memory");
    return r;
}

// rows of 16-bit features, `ld` bytes apart
struct Rows {
    const void* p;
    int64_t ld;
    __device__ __forceinline__ const char* row(uint32_t t) const { return static_cast<const char*>(p) + (uint64_t)ld * t; }
};
struct RowsTo {
    void* p;
    int64_t ld;
    bool aligned;  // 16-byte stores fit
    __device__ __forceinline__ char* row(uint32_t t) const { return static_cast<char*>(p) + (uint64_t)ld * t; }
};

__device__ __forceinline__ void copy16(uint32_t slot, const void* src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot), "l"(src), "r"(bytes) : "memory");
}

// The warp's features of a row into its piece of shared memory, asynchronously.
// Aligned rows: the lane's own 16 bytes of each half.  Others: the 16-byte chunks
// of memory that the features lie in, one more, whose other bytes are the row's
// (or the rows' beside it); the chunks that reach out of the tensor, in its first
// and last row, are read by the element.
template <bool ALIGNED>
__device__ __forceinline__ void fetch_row(uint32_t piece, const Rows& x, uint32_t t, uint32_t tokens, const Place& at)
{
    const char* row = x.row(t);
    if (ALIGNED) {  // piece: of the lane
        if (at.whole()) {
            asm volatile(
                "cp.async.cg.shared.global [%0], [%1], 16;\n\t"
                "cp.async.cg.shared.global [%0 + 512], [%1 + 512], 16;" ::"r"(piece), "l"(row + 2u * (uint32_t)at.first)
                : "memory");
        } else {
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const int have = at.have(h);
                copy16(piece + h * 512, row + (have > 0 ? 2 * (at.first + 256 * h) : 0), 2 * have);
            }
        }
        return;
    }
    const int lane = lane_id(), n = at.first + at.left;
    const char* from = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row + 2 * (at.first - lane * 8)) & ~(uintptr_t)15);
    const char *begin = static_cast<const char*>(x.p), *row_end = row + 2 * n, *end = x.row(tokens - 1) + 2 * n;
    for (int c = lane; c < 32 * kHalves + 1; c += 32) {
        const char* src = from + c * 16;
        if (src >= row_end) break;
        if (src >= begin && src + 16 <= end) {
            copy16(piece + c * 16, src, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (src + 2 * i >= begin && src + 2 * i < end)
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(piece + c * 16 + 2 * i), "h"(*reinterpret_cast<const unsigned short*>(src + 2 * i)) : "memory");
        }
    }
}

// the thread's features of that row; zero past its end
template <typename T, bool ALIGNED>
__device__ __forceinline__ Some row_at(uint32_t piece, const Rows& x, uint32_t t, const Place& at)
{
    if (ALIGNED) return packed_at<T>(piece);
    Some r;
    const int lane = lane_id();
    const uint32_t skew = (uint32_t)reinterpret_cast<uintptr_t>(x.row(t) + 2 * (at.first - lane * 8)) & 15u;  // bytes before the first feature
    const uint32_t from = piece + lane * 16 + (skew & ~3u);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        uint32_t u[5], w[4];
#pragma unroll
        for (int i = 0; i < 5; ++i)
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u[i]) : "r"(from + h * 512 + 4 * i) : "memory");
        const int have = at.have(h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __funnelshift_r(u[i], u[i + 1], 8 * (skew & 2u));
            if (have < 8) w[i] &= (2 * i < have ? 0xffffu : 0u) | (2 * i + 1 < have ? 0xffff0000u : 0u);
        }
        expand<T>(w, h, r);
    }
    return r;
}

// the thread's features into a row; rows that 16-byte stores do not fit go by way
// of `turn`, 512 bytes of the warp's own, so that a store covers 32 features in a row
template <typename T>
__device__ __forceinline__ void put(const RowsTo& out, uint32_t t, const Place& at, const Some& v, uint32_t turn)
{
    unsigned short* const row = reinterpret_cast<unsigned short*>(out.row(t) + 2 * at.first);
    const int lane = lane_id();
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = apart(v.v[4 * h + i]);
            w[i] = linear::pack2<T>(f.x, f.y);
        }
        unsigned short* p = row + 256 * h;
        const int left = at.left - 256 * h;
        if (out.aligned) {
            if (at.whole() || left >= 8) {
                *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < left) p[i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
            }
            continue;
        }
        __syncwarp();
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(turn + lane * 16), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        __syncwarp();
        p -= lane * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i * 32 + lane < left + lane * 8) {
                unsigned short e;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(e) : "r"(turn + 2 * (i * 32 + lane)) : "memory");
                p[i * 32 + lane] = e;
            }
    }
}

// ----------------------------------------------------------------------------
// sums over a row
// ----------------------------------------------------------------------------
template <int LANES = 32>
__device__ __forceinline__ float warp_sum(float a)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) a += __shfl_xor_sync(0xffffffffu, a, d);
    return a;
}

// Sums over the row of a group; every thread of it calls with the same calls
// before.  Warps' sums go through shared memory, two sets of them in turn: who
// writes a set again has passed the barrier that all readers of its last use
// reached afterwards.  Where a cluster shares the row every warp sends its sums to
// all CTAs of it, and arrives there on the group's own barrier: groups do not wait
// for one another.
struct WarpSums {
    float2 of[2][kClusterGroups][kMaxWarps + 1];  // the last one stays zero
    uint64_t bar[2][kClusterGroups];
    int gave_up;
};

__device__ int g_status;  // sticky device-side error of this module

// eight bytes to a CTA of the cluster, counted on its barrier.  (A release at
// cluster scope beside plain stores would wait for the rows' stores under way: a
// row of 16384 features took 1.7 times as long.)
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, float a, float b)
{
    const Two v = two(a, b);
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(v.v), "r"(bar) : "memory");
}

struct RowSums {
    uint32_t mine, from;  // where the warp puts its sums, and where a lane reads one (or the zero)
    uint64_t* bar;        // of the group
    bool leads;           // its first warp
    bool few;             // up to eight warps share the row: every eight lanes read all of their sums
    int warps, group, cluster;
    uint32_t set, phase;  // of the next use; the barriers' parity
    volatile int* gave_up;

    __device__ __forceinline__ RowSums(WarpSums& sets, const Shape& s, int of_group)
        : warps(s.warps), group(of_group), cluster(s.cluster), set(0), phase(0), gave_up(&sets.gave_up)
    {
        const int lane = lane_id(), warp = warp_id() - group * warps;
        const int row = cluster > 1 ? group : 0, first = cluster > 1 ? (int)cluster_ctarank() * warps : group * warps;
        mine = smem_u32(&sets.of[0][row][first + warp]);
        few = cluster * warps <= 8;
        const int entry = few ? lane % 8 : lane;
        from = smem_u32(&sets.of[0][row][entry < cluster * warps ? (cluster > 1 ? 0 : first) + entry : kMaxWarps]);
        bar = &sets.bar[0][row];
        leads = warp == 0;
        if (threadIdx.x < 2 * kClusterGroups) {
            sets.of[threadIdx.x / kClusterGroups][threadIdx.x % kClusterGroups][kMaxWarps] = make_float2(0.0f, 0.0f);
            mbar_init(&sets.bar[threadIdx.x / kClusterGroups][threadIdx.x % kClusterGroups], 1);
            fence_barrier_init();
        }
        if (threadIdx.x == 0) sets.gave_up = 0;
        if (cluster > 1) cluster_sync();
        else __syncthreads();
    }
    __device__ __forceinline__ float2 exchange(float a, float b)
    {
        const uint32_t other = set ? (uint32_t)sizeof(WarpSums::of[0]) : 0u;
        if (cluster == 1) {
            if (lane_id() == 0) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(mine + other), "f"(a), "f"(b) : "memory");
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * warps) : "memory");
        } else {
            uint64_t* at = bar + set * kClusterGroups;
            if (leads && lane_id() == 0) mbar_arrive_expect_tx(at, cluster * warps * 8);
            if (lane_id() < cluster) send(map_to_rank(mine + other, lane_id()), map_to_rank(smem_u32(at), lane_id()), a, b);
            if (!mbar_wait(at, phase, gave_up)) atomicExch(&g_status, CHPL_ERR_TIMEOUT);
            __syncwarp();
            phase ^= set;
        }
        float2 v;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(from + other) : "memory");
        set ^= 1u;
        return v;
    }
    __device__ __forceinline__ float one(float a)
    {
        a = warp_sum(a);
        if (warps * cluster == 1) return a;
        a = exchange(a, 0.0f).x;
        return few ? warp_sum<8>(a) : warp_sum(a);
    }
    __device__ __forceinline__ float2 both_of(float a, float b)
    {
        a = warp_sum(a);
        b = warp_sum(b);
        if (warps * cluster == 1) return make_float2(a, b);
        const float2 v = exchange(a, b);
        return few ? make_float2(warp_sum<8>(v.x), warp_sum<8>(v.y)) : make_float2(warp_sum(v.x), warp_sum(v.y));
    }
};

// The rows under way: copies of the rows to come, a group of cp.async each,
// `stages` of them (an empty group where there is no such row).  Aligned rows' pieces
// start on 128 bytes: 16 bytes off a line the copies ask L2 for 1.6 times the bytes
// and a join of 8192 x 4096 takes 53 us instead of 47.4, its gradients 84 instead of
// 73.5.
struct Ring {
    uint32_t tensor, bytes, end;  // between tensors, of a stage, behind the last one
    uint32_t at;                  // the warp's (the lane's, where rows are aligned) piece of the current row's first tensor
    int stages;
    __device__ __forceinline__ Ring(uint32_t mine, int tensors, const Shape& s)
        : tensor((blockDim.x >> 5) * s.piece), bytes(tensors * tensor), end(mine + s.stages * bytes), at(mine), stages(s.stages)
    {
    }
    __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // the oldest of `stages` groups has arrived, the whole warp's where a lane reads others' copies
    template <bool ALIGNED>
    __device__ __forceinline__ void wait() const
    {
        static_assert(kMaxStages == 2, "the groups waited for");
        if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (!ALIGNED) __syncwarp();
    }
    __device__ __forceinline__ void next()
    {
        at += bytes;
        if (at == end) at -= stages * bytes;
    }
};

// ----------------------------------------------------------------------------
// forward
// ----------------------------------------------------------------------------
struct Forward {
    uint32_t tokens;
    int n;
    float scale, residual_scale, post_eps, pre_eps;
    int post, pre;          // kinds
    Rows x, y, gate;        // gate.ld 0: a vector
    const void *post_w, *post_b, *pre_w, *pre_b;
    RowsTo r, h;
    float2 *post_stats, *pre_stats;
};

// (v - mean) / deviation, w v + b of it; (mean, 1 / deviation) to *stats.  Mean
// first, then the squares of what is left: the one pass of squares loses the
// variance of rows whose mean is large.
__device__ __forceinline__ Some normalize(Some v, const Place& at, int kind, float eps, float inv_n, uint32_t w, uint32_t b, bool has_b,
                                          RowSums& sums, float2* stats, bool writes)
{
    float mean = 0.0f;
    if (kind == CHPL_NORM_LAYER) {
        mean = sums.one(total_of(v)) * inv_n;  // zero past the end
        v = v + -mean;
        if (!at.whole()) clear_tail(v, at);
    }
    const float rstd = rsqrtf(fmaf(sums.one(dot(v, v)), inv_n, eps));
    if (stats && writes) *stats = make_float2(mean, rstd);
    v = v * rstd;
    return has_b ? fma_of(v, vector_at(w), vector_at(b)) : v * vector_at(w);
}

template <typename T, bool ALIGNED, bool JOIN>
__global__ void __launch_bounds__(kForwardThreads) forward_kernel(const __grid_constant__ Forward a, const Shape s)
{
    extern __shared__ __align__(128) uint4 smem[];
    __shared__ WarpSums sets;
    const Place at(s, a.n);
    const bool matrix = JOIN && a.gate.p && a.gate.ld;
    const int tensors = JOIN ? 2 + matrix : 1;
    const uint32_t mem = smem_u32(smem), vec = mem + (warp_id() - at.group * s.warps) * kVectorBytes + lane_id() * 16, vec_step = s.warps * kVectorBytes,
                   turn = mem + s.turn + warp_id() * 512;
    // the vectors that there are, then the rows; a vector gate and the scale are in post_w and post_b
    uint32_t used = 0;
    const auto place = [&](bool there) { return vec + (there ? used++ : 0) * vec_step; };
    const bool weighs = JOIN && (a.post || (a.gate.p && !matrix));
    const uint32_t pre_w = place(a.pre), pre_b = place(a.pre_b), post_w = JOIN ? place(weighs) : 0, post_b = JOIN ? place(a.post_b) : 0;
    Ring ring(mem + used * vec_step + warp_id() * s.piece + (ALIGNED ? lane_id() * 16 : 0), tensors, s);
    RowSums sums(sets, s, at.group);
    const float inv_n = 1.0f / (float)a.n;
    start_of_inputs();
    const auto load = [&](uint32_t row, uint32_t slot) {
        if (row < a.tokens) {
            fetch_row<ALIGNED>(slot + 0 * ring.tensor, a.x, row, a.tokens, at);
            if (JOIN) fetch_row<ALIGNED>(slot + 1 * ring.tensor, a.y, row, a.tokens, at);
            if (JOIN && matrix) fetch_row<ALIGNED>(slot + 2 * ring.tensor, a.gate, row, a.tokens, at);
        }
        Ring::commit();
    };
    for (int i = 0; i < s.stages; ++i) load(at.row + i * at.step, ring.at + i * ring.bytes);
    if (at.group == 0) {  // the groups' in common
        const Raw<T> none = raw_vector<T>(nullptr, false, at), w1 = raw_vector<T>(a.pre_w, a.pre, at), b1 = raw_vector<T>(a.pre_b, a.pre_b, at);
        if (JOIN) {
            const Raw<T> w0 = raw_vector<T>(a.post_w, a.post, at), b0 = raw_vector<T>(a.post_b, a.post_b, at),
                         g0 = raw_vector<T>(a.gate.p, a.gate.p && !matrix, at);
            if (weighs) put_vector<T>(post_w, w0, g0, a.scale);
            if (a.post_b) put_vector<T>(post_b, b0, g0, a.scale);
        }
        if (a.pre) put_vector<T>(pre_w, w1, none, 1.0f);
        if (a.pre_b) put_vector<T>(pre_b, b1, none, 1.0f);
    }
    __syncthreads();
    const bool writes = at.first == 0;  // the row's statistics
    for (uint32_t row = at.row; row < a.tokens; row += at.step, ring.next()) {
        ring.template wait<ALIGNED>();
        Some v;
        if (JOIN) {
            v = row_at<T, ALIGNED>(ring.at + 1 * ring.tensor, a.y, row, at);
            if (a.post)
                v = normalize(v, at, a.post, a.post_eps, inv_n, post_w, post_b, a.post_b, sums, a.post_stats ? a.post_stats + row : nullptr, writes);
            else
                v = weighs ? v * vector_at(post_w) : v * a.scale;
            if (matrix) v = v * row_at<T, ALIGNED>(ring.at + 2 * ring.tensor, a.gate, row, at);
            v = fma_of(row_at<T, ALIGNED>(ring.at + 0 * ring.tensor, a.x, row, at), a.residual_scale, v);
            put<T>(a.r, row, at, v, turn);
        } else {
            v = row_at<T, ALIGNED>(ring.at + 0 * ring.tensor, a.x, row, at);
        }
        if (!ALIGNED) __syncwarp();
        load(row + s.stages * at.step, ring.at);
        if (a.pre) {
            v = normalize(v, at, a.pre, a.pre_eps, inv_n, pre_w, pre_b, a.pre_b, sums, a.pre_stats ? a.pre_stats + row : nullptr, writes);
            put<T>(a.h, row, at, v, turn);
        }
    }
    if (s.cluster > 1) cluster_sync();  // no CTA leaves while another still sends to it
}

// ----------------------------------------------------------------------------
// backward
// ----------------------------------------------------------------------------
// What a join has, known to the kernel where its rows are aligned (PARTS < 0: it
// looks).  Straight code, without branches around what is not there: 8192 x 4096 with
// two RMS norms 95 -> 89 us.  (The forward kernel gains nothing by it.)
enum { kPre = 1, kPost = 2, kMatrix = 4, kAnyParts = -1 };
template <int PARTS>
__device__ __forceinline__ bool part(int which, bool there)
{
    return PARTS < 0 ? there : (PARTS & which) != 0;
}

struct Backward {
    uint32_t tokens;
    int n;
    float scale, residual_scale;
    int post, pre;
    Rows dr, dh, r, y, gate;  // gate.ld 0: a vector; y.p NULL: not wanted
    const void *post_w, *post_b, *pre_w;
    const float2 *post_stats, *pre_stats;
    RowsTo dx, dy, dgate;     // dgate of a matrix
    float* part;              // [sum][unit][part_ld] of the sums that `sums` names
    int part_ld;              // n, up to a multiple of four
    int sums;                 // bit k: sum k
};

// Sums over the tokens, from which the parameters' gradients follow: with Do =
// alpha D (times the gate where it is a matrix), yhat the normed y (or y),
//   0  Do yhat   dw_post = gate * 0,  dgate = w_post * 0 + b_post * 1
//   1  Do        db_post = gate * 1
//   2  dh rhat   dw_pre
//   3  dh        db_pre
constexpr int kSums = 4;

// With c = v - m the gradient of a norm at v is s (g - mean(g) - c s^2 mean(g c)),
// g = d weight: g s, mean(g s) and mean(g s c) are formed, which takes one product
// an element less than the normed value would.  Rows' tails, which the copies leave
// zero, need no masks: every sum over the row has a factor of a zero weight.
struct Pull {
    float mean, along;  // what is taken off: mean + along c
};
__device__ __forceinline__ Pull pull(const Some& g, const Some& c, int kind, float s, float inv_n, RowSums& sums)
{
    if (kind != CHPL_NORM_LAYER) return {0.0f, sums.one(dot(g, c)) * inv_n * s * s};
    const float2 t = sums.both_of(total_of(g), dot(g, c));
    return {t.x * inv_n, t.y * inv_n * s * s};
}

template <typename T, bool ALIGNED, bool JOIN, bool BIAS, int PARTS>
__global__ void __launch_bounds__(kBackwardThreads) backward_kernel(const __grid_constant__ Backward a, const Shape s)
{
    const bool has_pre = part<PARTS>(kPre, a.pre), has_post = JOIN && part<PARTS>(kPost, a.post);
    extern __shared__ __align__(128) uint4 smem[];
    __shared__ WarpSums sets;
    const Place at(s, a.n);
    const bool matrix = JOIN && part<PARTS>(kMatrix, a.gate.p && a.gate.ld), has_y = JOIN && (has_post || a.y.p), weighs = JOIN && (has_post || (a.gate.p && !matrix));
    const int t_dh = 0, t_r = 1, t_y = has_pre ? 2 : 0, t_gate = t_y + has_y, t_dr = t_gate + matrix, tensors = t_dr + (a.dr.p ? 1 : 0);
    const uint32_t mem = smem_u32(smem), vec = mem + (warp_id() - at.group * s.warps) * kVectorBytes + lane_id() * 16, vec_step = s.warps * kVectorBytes,
                   turn = mem + s.turn + warp_id() * 512;
    uint32_t used = 0;  // a vector gate is in post_w
    const auto place = [&](bool there) { return vec + (there ? used++ : 0) * vec_step; };
    const uint32_t pre_w = place(has_pre), post_w = JOIN ? place(weighs) : 0, post_b = JOIN ? place(matrix && a.post_b) : 0;
    Ring ring(mem + used * vec_step + warp_id() * s.piece + (ALIGNED ? lane_id() * 16 : 0), tensors, s);
    RowSums sums(sets, s, at.group);
    const float inv_n = 1.0f / (float)a.n;
    const auto of = [&](int t, const Rows& x, uint32_t row) { return row_at<T, ALIGNED>(ring.at + t * ring.tensor, x, row, at); };
    start_of_inputs();
    const auto load = [&](uint32_t row, uint32_t slot) {
        if (row < a.tokens) {
            const auto fetch = [&](int t, const Rows& x) { fetch_row<ALIGNED>(slot + t * ring.tensor, x, row, a.tokens, at); };
            if (a.dr.p) fetch(t_dr, a.dr);
            if (has_pre) {
                fetch(t_dh, a.dh);
                fetch(t_r, a.r);
            }
            if (has_y) fetch(t_y, a.y);
            if (matrix) fetch(t_gate, a.gate);
        }
        Ring::commit();
    };
    const auto stats_of = [&](uint32_t row, float2& pre, float2& post) {
        pre = post = make_float2(0.0f, 1.0f);
        if (row >= a.tokens) return;
        if (has_pre) pre = __ldg(a.pre_stats + row);
        if (has_post) post = __ldg(a.post_stats + row);
    };
    for (int i = 0; i < s.stages; ++i) load(at.row + i * at.step, ring.at + i * ring.bytes);
    if (at.group == 0) {  // the groups' in common
        const Raw<T> none = raw_vector<T>(nullptr, false, at), w1 = raw_vector<T>(a.pre_w, has_pre, at);
        if (JOIN) {
            const Raw<T> w0 = raw_vector<T>(a.post_w, has_post, at), b0 = raw_vector<T>(a.post_b, matrix && a.post_b, at),
                         g0 = raw_vector<T>(a.gate.p, a.gate.p && !matrix, at);
            if (weighs) put_vector<T>(post_w, w0, g0, 1.0f);
            if (matrix && a.post_b) put_vector<T>(post_b, b0, none, 1.0f);
        }
        if (has_pre) put_vector<T>(pre_w, w1, none, 1.0f);
    }
    __syncthreads();
    constexpr int kTotals = (BIAS ? 2 : 1) * (JOIN ? 2 : 1);  // without a join sums 2 and 3, without biases 0 and 2
    constexpr int kHat = JOIN ? (BIAS ? 2 : 1) : 0;
    Some total[kTotals];
#pragma unroll
    for (int k = 0; k < kTotals; ++k) total[k] = zeros();
    float2 pre_next, post_next;
    stats_of(at.row, pre_next, post_next);
    for (uint32_t row = at.row; row < a.tokens; row += at.step, ring.next()) {
        const float2 pre = pre_next, post = post_next;
        stats_of(row + at.step, pre_next, post_next);
        ring.template wait<ALIGNED>();
        Some d;
        if (has_pre) {
            Some c = of(t_r, a.r, row), g = of(t_dh, a.dh, row);
            if constexpr (BIAS) total[kHat + 1] = total[kHat + 1] + g;
            if (a.pre == CHPL_NORM_LAYER) c = c + -pre.x;
            g = g * pre.y;
            total[kHat] = fma_of(g, c, total[kHat]);
            g = g * vector_at(pre_w);
            const Pull p = pull(g, c, a.pre, pre.y, inv_n, sums);
            d = fma_of(c, -p.along, g);
            if (a.pre == CHPL_NORM_LAYER) d = d + -p.mean;
            if (a.dr.p) d = d + of(t_dr, a.dr, row);
        } else {
            d = of(t_dr, a.dr, row);
        }
        if (a.dx.p) put<T>(a.dx, row, at, JOIN ? d * a.residual_scale : d, turn);
        if (JOIN) {
            Some y = zeros();
            if (has_y) y = of(t_y, a.y, row);
            if (a.post == CHPL_NORM_LAYER) y = y + -post.x;
            // Do, times 1 / deviation of y
            if (BIAS) d = d * a.scale;
            if (matrix) {
                if (a.dgate.p) {
                    Some p = y * post.y;
                    if (has_post) p = a.post_b ? fma_of(p, vector_at(post_w), vector_at(post_b)) : p * vector_at(post_w);
                    put<T>(a.dgate, row, at, (BIAS ? d : d * a.scale) * p, turn);
                }
                d = d * of(t_gate, a.gate, row);
            }
            if constexpr (BIAS) total[1] = total[1] + d;
            d = d * (BIAS ? post.y : post.y * a.scale);
            total[0] = fma_of(d, y, total[0]);
            if (weighs) d = d * vector_at(post_w);
            if (!ALIGNED) __syncwarp();
            load(row + s.stages * at.step, ring.at);
            if (has_post) {
                const Pull p = pull(d, y, a.post, post.y, inv_n, sums);
                d = fma_of(y, -p.along, d);
                if (a.post == CHPL_NORM_LAYER) d = d + -p.mean;
            }
            if (a.dy.p) put<T>(a.dy, row, at, d, turn);
        } else {
            if (!ALIGNED) __syncwarp();
            load(row + s.stages * at.step, ring.at);
        }
    }
    // A CTA's sums: every thread's into shared memory, where the rows under way were,
    // then all threads add up the groups', in order, four features at a time.
    if (a.part) {
        const int quads = s.warps * (kWarpWidth / 4);  // of a group
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        uint32_t put_at = mem + ((warp_id() - at.group * s.warps) * (kWarpWidth / 4) + lane_id()) * 16 + at.group * quads * 16;
        int count = 0;
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            if ((!JOIN && k < 2) || (!BIAS && k % 2)) continue;
            if (!(a.sums >> k & 1)) continue;
            const Some& mine = total[BIAS ? k - (JOIN ? 0 : 2) : JOIN ? k / 2 : 0];
#pragma unroll
            for (int i = 0; i < kTwos; i += 2)  // quad i / 2 of the lane's
                asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(put_at + i * 256), "l"(mine.v[i].v), "l"(mine.v[i + 1].v) : "memory");
            put_at += s.groups * quads * 16;
            ++count;
        }
        __syncthreads();
        const int rank = s.cluster > 1 ? (int)cluster_ctarank() : 0;
        const int64_t unit = blockIdx.x / s.cluster;
        for (int i = threadIdx.x; i < count * quads; i += blockDim.x) {
            const int k = i / quads, q = i - k * quads, warp = q / (kWarpWidth / 4), in = q % (kWarpWidth / 4);
            // the in-th four of the warp's features: quad in % 2 of half in / 64 of lane in / 2 % 32
            const uint32_t from = mem + (uint32_t)(((k * s.groups * s.warps + warp) * (kWarpWidth / 4) + (in / 64 * 2 + in % 2) * 32 + in / 2 % 32) * 16);
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int g = 0; g < s.groups; ++g) {
                float4 v;
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(from + g * quads * 16) : "memory");
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            const int j = (rank * s.warps + warp) * kWarpWidth + in * 4;
            if (j < a.n) *reinterpret_cast<float4*>(a.part + ((int64_t)k * s.units + unit) * a.part_ld + j) = sum;  // past n: padding
        }
    }
    if (s.cluster > 1) cluster_sync();
}

// The parameters' gradients from the units' sums.  A block takes 32 features, its
// warps equal runs of the units, joined in order; bound by the loads' latency.
struct Parameters {
    const float* part;
    int part_ld, units, n, sums;
    int f32, accumulate, matrix;
    const void *post_w, *post_b, *gate;  // as they were used
    void *dpost_w, *dpost_b, *dgate, *dpre_w, *dpre_b;
};

constexpr int kJoinWarps = 32;  // at most: one to four units

template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) parameters_kernel(const __grid_constant__ Parameters a)
{
    __shared__ float turn[kSums][kJoinWarps][32];
    const int lane = lane_id(), warp = warp_id(), warps = blockDim.x / 32, j = blockIdx.x * 32 + lane;
    const int first = (int)((int64_t)a.units * warp / warps), last = (int)((int64_t)a.units * (warp + 1) / warps);
    const int count = __popc(a.sums);
    const int64_t step = (int64_t)a.units * a.part_ld;  // from one sum to the next
    start_of_inputs();
    const auto of = [&](const void* v, float other) { return v && j < a.n ? to_f32(static_cast<const T*>(v)[j]) : other; };
    float gate = 1.0f, weight = 1.0f, bias = 0.0f;
    if (warp == 0) {
        gate = a.matrix ? 1.0f : of(a.gate, 1.0f);  // a matrix is in the sums
        weight = of(a.post_w, 1.0f);
        bias = of(a.post_b, 0.0f);
    }
    float sum[kSums] = {};
    if (j < a.n) {
        const float* p = a.part + j;
#pragma unroll 4
        for (int u = first; u < last; ++u)
#pragma unroll
            for (int c = 0; c < kSums; ++c)
                if (c < count) sum[c] += p[c * step + (int64_t)u * a.part_ld];
    }
#pragma unroll
    for (int c = 0; c < kSums; ++c) turn[c][warp][lane] = sum[c];
    __syncthreads();
    if (warp > 0 || j >= a.n) return;
    float all[kSums] = {};
    int slot = 0;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        if (!(a.sums >> k & 1)) continue;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) all[k] += turn[slot][w][lane];
        ++slot;
    }
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
    store(a.dpost_w, gate * all[0]);
    store(a.dpost_b, gate * all[1]);
    store(a.dgate, a.post_b ? fmaf(weight, all[0], bias * all[1]) : weight * all[0]);
    store(a.dpre_w, all[2]);
    store(a.dpre_b, all[3]);
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

// 16-byte accesses fit
static bool fits(const void* p, int64_t ld, int64_t tokens) { return !p || aligned(p, tokens > 1 ? ld * 2 : 0, 16); }

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
    CHPL_TRY(allow_smem(KERNEL, kSmem - kSmemApart, ready));
    return launch_kernel(KERNEL, (int64_t)s.units * s.cluster, 32 * s.warps * s.groups, s.smem, s.cluster, st, a, s);
}

// what a forward call is launched as
struct ForwardPlan {
    Shape shape;
    bool in;  // rows that 16-byte accesses fit
};

static ForwardPlan plan(const chpl_norm_fwd& a)
{
    const bool post = a.join && a.post.kind, matrix = a.join && a.gate && a.ldgate;
    ForwardPlan p;
    p.in = fits(a.x, a.ldx, a.tokens) && (!a.join || fits(a.y, a.ldy, a.tokens)) && (!matrix || fits(a.gate, a.ldgate, a.tokens));
    const bool out = (!a.join || fits(a.r, a.ldr, a.tokens)) && (!a.pre.kind || fits(a.h, a.ldh, a.tokens));
    const int vectors = (a.pre.kind ? 1 + (a.pre.bias != nullptr) : 0) + (post || (a.join && a.gate && !matrix) ? 1 : 0) + (post && a.post.bias ? 1 : 0);
    p.shape = shape_for(a.tokens, a.n, a.join ? 2 + matrix : 1, vectors, p.in, out, kForwardThreads);
    return p;
}

template <typename T>
static int forward(cudaStream_t st, const chpl_norm_fwd& a)
{
    const ForwardPlan p = plan(a);
    Forward f = {};
    f.tokens = (uint32_t)a.tokens;
    f.n = (int)a.n;
    f.scale = a.scale;
    f.residual_scale = a.residual_scale;
    f.x = {a.x, a.ldx * 2};
    if (a.join) {
        f.post = a.post.kind;
        f.post_eps = a.post.eps;
        f.y = {a.y, a.ldy * 2};
        f.gate = {a.gate, a.ldgate * 2};
        f.r = {a.r, a.ldr * 2, fits(a.r, a.ldr, a.tokens)};
        if (f.post) {
            f.post_w = a.post.weight;
            f.post_b = a.post.bias;
            f.post_stats = reinterpret_cast<float2*>(a.post_stats);
        }
    }
    f.pre = a.pre.kind;
    if (f.pre) {
        f.pre_eps = a.pre.eps;
        f.pre_w = a.pre.weight;
        f.pre_b = a.pre.bias;
        f.h = {a.h, a.ldh * 2, fits(a.h, a.ldh, a.tokens)};
        f.pre_stats = reinterpret_cast<float2*>(a.pre_stats);
    }
    if (a.join) return p.in ? launch<forward_kernel<T, true, true>>(st, f, p.shape) : launch<forward_kernel<T, false, true>>(st, f, p.shape);
    return p.in ? launch<forward_kernel<T, true, false>>(st, f, p.shape) : launch<forward_kernel<T, false, false>>(st, f, p.shape);
}

// what a backward call forms
struct BackwardPlan {
    Shape shape;
    bool in, out;    // rows that 16-byte accesses fit
    int sums;        // bits
    int part_ld;
    size_t bytes;
};

// y, or what is left of it after its mean, is a factor of the norm's gradients and of the gate's
static bool wants_y(const chpl_norm_bwd& a) { return a.join && (a.post.kind || a.dgate); }

static BackwardPlan plan(const chpl_norm_bwd& a)
{
    BackwardPlan p;
    const bool vector_gate = a.dgate && a.gate && a.ldgate == 0, matrix = a.join && a.gate && a.ldgate, has_y = wants_y(a);
    p.sums = 0;
    if (a.join && ((a.post.kind && a.dpost_weight) || vector_gate)) p.sums |= 1;
    if (a.join && a.post.kind && (a.dpost_bias || (vector_gate && a.post.bias))) p.sums |= 2;
    if (a.pre.kind && a.dpre_weight) p.sums |= 4;
    if (a.pre.kind && a.dpre_bias) p.sums |= 8;
    p.in = fits(a.dr, a.lddr, a.tokens) && (!a.pre.kind || (fits(a.dh, a.lddh, a.tokens) && fits(a.r, a.ldr, a.tokens))) &&
           (!has_y || fits(a.y, a.ldy, a.tokens)) && (!matrix || fits(a.gate, a.ldgate, a.tokens));
    p.out = fits(a.dx, a.lddx, a.tokens) && (!a.join || fits(a.dy, a.lddy, a.tokens)) && (!matrix || fits(a.dgate, a.lddgate, a.tokens));
    const int tensors = (a.dr ? 1 : 0) + (a.pre.kind ? 2 : 0) + has_y + matrix;
    const int vectors = (a.pre.kind ? 1 : 0) + (a.join && (a.post.kind || (a.gate && a.ldgate == 0)) ? 1 : 0) + (matrix && a.post.kind && a.post.bias ? 1 : 0);
    p.shape = shape_for(a.tokens, a.n, tensors, vectors, p.in, p.out, kBackwardThreads);
    int count = 0;
    for (int k = 0; k < kSums; ++k) count += p.sums >> k & 1;
    // the groups' sums are joined where the rows under way were
    p.shape.smem = std::max(p.shape.smem, count * kWarpWidth * p.shape.warps * p.shape.groups * 4);
    p.part_ld = (int)round_up((size_t)a.n, 4);
    // as many units as any launch of so many tokens has (fewer where a CTA holds several rows or shares one), so that
    // what serves a batch serves every smaller one, wherever its operands lie
    p.bytes = round_up((size_t)count * std::min<int64_t>(a.tokens, kSms) * p.part_ld * 4, 256);
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
        if (wants_y(*a)) CHPL_TRY(check_operand(who, "y", a->y, a->ldy, a->n, 2));
        if (a->post.kind) CHPL_TRY(check_stats(who, "statistics of y", a->post_stats, true));
        if (a->dy) CHPL_TRY(check_operand(who, "dy", a->dy, a->lddy, a->n, 2));
        if (a->dgate && a->ldgate) CHPL_TRY(check_operand(who, "dgate", a->dgate, a->lddgate, a->n, 2));
    }
    return CHPL_OK;
}

static int parts_of(const chpl_norm& pre, const chpl_norm& post, const void* gate, int64_t ldgate)
{
    return (pre.kind ? kPre : 0) | (post.kind ? kPost : 0) | (gate && ldgate ? kMatrix : 0);
}

template <int V>
struct Parts {
    static constexpr int value = V;
};
template <typename F>
static int with_parts(int parts, F&& f)
{
    switch (parts) {
        case 0: return f(Parts<0>());
        case 1: return f(Parts<1>());
        case 2: return f(Parts<2>());
        case 3: return f(Parts<3>());
        case 4: return f(Parts<4>());
        case 5: return f(Parts<5>());
        case 6: return f(Parts<6>());
        default: return f(Parts<7>());
    }
}

template <typename T, bool BIAS>
static int launch_backward(cudaStream_t st, const chpl_norm_bwd& a, const Backward& b, const BackwardPlan& p)
{
    if (!a.join)
        return p.in ? launch<backward_kernel<T, true, false, BIAS, kPre>>(st, b, p.shape) : launch<backward_kernel<T, false, false, BIAS, kPre>>(st, b, p.shape);
    if (!p.in) return launch<backward_kernel<T, false, true, BIAS, kAnyParts>>(st, b, p.shape);
    return with_parts(parts_of(a.pre, a.post, a.gate, a.ldgate),
                      [&](auto parts) { return launch<backward_kernel<T, true, true, BIAS, decltype(parts)::value>>(st, b, p.shape); });
}

template <typename T>
static int backward(cudaStream_t st, const chpl_norm_bwd& a, void* work)
{
    const BackwardPlan p = plan(a);
    const bool matrix = a.join && a.gate && a.ldgate;
    if (a.tokens > 0) {
        Backward b = {};
        b.tokens = (uint32_t)a.tokens;
        b.n = (int)a.n;
        b.scale = a.scale;
        b.residual_scale = a.residual_scale;
        b.sums = p.sums;
        b.part = p.sums ? static_cast<float*>(work) : nullptr;
        b.part_ld = p.part_ld;
        b.dr = {a.dr, a.lddr * 2};
        b.dx = {a.dx, a.lddx * 2, fits(a.dx, a.lddx, a.tokens)};
        if (a.pre.kind) {
            b.pre = a.pre.kind;
            b.dh = {a.dh, a.lddh * 2};
            b.r = {a.r, a.ldr * 2};
            b.pre_w = a.pre.weight;
            b.pre_stats = reinterpret_cast<const float2*>(a.pre_stats);
        }
        if (a.join) {
            if (wants_y(a)) b.y = {a.y, a.ldy * 2};
            b.gate = {a.gate, a.ldgate * 2};
            b.dy = {a.dy, a.lddy * 2, fits(a.dy, a.lddy, a.tokens)};
            if (matrix) b.dgate = {a.dgate, a.lddgate * 2, fits(a.dgate, a.lddgate, a.tokens)};
            if (a.post.kind) {
                b.post = a.post.kind;
                b.post_w = a.post.weight;
                b.post_b = a.post.bias;
                b.post_stats = reinterpret_cast<const float2*>(a.post_stats);
            }
        }
        const bool bias = (p.sums & 10) != 0;
        CHPL_TRY((bias ? launch_backward<T, true>(st, a, b, p) : launch_backward<T, false>(st, a, b, p)));
    }
    if (!p.sums || (a.tokens == 0 && a.accumulate)) return CHPL_OK;
    Parameters q = {};
    q.part = static_cast<const float*>(work);
    q.part_ld = p.part_ld;
    q.units = a.tokens > 0 ? p.shape.units : 0;
    q.n = (int)a.n;
    q.sums = p.sums;
    q.f32 = a.grad_type == CHPL_TYPE_F32;
    q.accumulate = a.accumulate;
    q.matrix = matrix;
    const bool any = a.tokens > 0;  // without tokens sums of nothing, not 0 times what a gate or a weight may hold
    if (a.join) {
        if (any) q.gate = a.gate;
        if (!matrix) q.dgate = a.dgate;
        if (a.post.kind) {
            if (any) q.post_w = a.post.weight;
            if (any) q.post_b = a.post.bias;
            q.dpost_w = a.dpost_weight;
            q.dpost_b = a.dpost_bias;
        }
    }
    if (a.pre.kind) {
        q.dpre_w = a.dpre_weight;
        q.dpre_b = a.dpre_bias;
    }
    return launch_kernel(parameters_kernel<T>, (a.n + 31) / 32, 32 * std::max(1, std::min(kJoinWarps, (q.units + 3) / 4)), 0, 1, st, q);
}

static void describe(const Shape& s, int64_t plan[3])
{
    plan[0] = s.cluster;
    plan[1] = s.groups;
    plan[2] = s.units;
}

int read_clear_status(int* st)
{
    int v = 0, z = 0;
    CHPL_CUDA(cudaMemcpyFromSymbol(&v, g_status, sizeof(int)));
    CHPL_CUDA(cudaMemcpyToSymbol(g_status, &z, sizeof(int)));
    *st = v;
    return CHPL_OK;
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

extern "C" int chpl_diag_norm_forward_plan(const chpl_norm_fwd* a, int64_t plan[3])
{
    const char* who = "diag_norm_forward_plan";
    CHPL_TRY(chpl::norm::check(who, a));
    if (!plan || !a->tokens || !a->n) { chpl::set_error("%s: nothing to plan", who); return CHPL_ERR_INVALID; }
    chpl::norm::describe(chpl::norm::plan(*a).shape, plan);
    return CHPL_OK;
}

extern "C" int chpl_diag_norm_backward_plan(const chpl_norm_bwd* a, int64_t plan[3])
{
    const char* who = "diag_norm_backward_plan";
    CHPL_TRY(chpl::norm::check(who, a, true));
    if (!plan || !a->tokens || !a->n) { chpl::set_error("%s: nothing to plan", who); return CHPL_ERR_INVALID; }
    chpl::norm::describe(chpl::norm::plan(*a).shape, plan);
    return CHPL_OK;
}
