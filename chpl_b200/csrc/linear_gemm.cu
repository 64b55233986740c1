// The linear-layer products on the tensor cores: D[f][t] = sum_c A(f, c) B(t, c)
// with the epilogue of linear_epilogue.cuh.
//
// Every product is oriented so that the output's contiguous dimension f (the
// features) lies along the 128 TMEM lanes and its rows t along the columns: a
// checkpoint group of 32 features is one warp's lanes, and a few tokens fill a
// narrow tile (t is the MMA's N dimension, 16 to 256) instead of a fraction of
// a 128-row one.
//
//   forward      A = W (c contiguous)      B = X (c contiguous)
//   grad input   A = W^T (f contiguous)    B = G (c contiguous)
//   grad weight  A = Xv^T (f contiguous)   B = G^T (t contiguous)
//
// Operands whose contiguous dimension is c are K-major for tcgen05.mma, the
// others MN-major; both come by TMA as 128-byte swizzled boxes 64 elements
// wide, zero beyond the matrix, so no size needs padding.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "linear_epilogue.cuh"

namespace chpl {
namespace linear {

__device__ int g_status;  // sticky device-side error of this module

constexpr int BM = 128;               // features of a tile (TMEM lanes)
constexpr int BK = 64;                // contraction elements of a stage: 128 bytes
constexpr int UK = 16;                // contraction elements of one MMA
constexpr int A_BYTES = BM * BK * 2;  // one stage of A
constexpr int BOX_BYTES = 64 * BK * 2;  // a 64-wide MN-major box
constexpr int MAX_STAGES = 12;
constexpr int SMEM_LIMIT = 227 * 1024;

// ----------------------------------------------------------------------------
// tcgen05 kind::f16 (bf16 / f16 operands, FP32 accumulators)
// ----------------------------------------------------------------------------
// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: rows of 128
// bytes, 8-row groups 1024 bytes apart (stride offset; the leading offset is
// not used).  MN-major: 64 elements of M or N per 128-byte row, c down the
// rows in groups of 8 that are 1024 bytes apart (stride offset), the next 64
// of M or N one box further (leading offset).
//
// The high word is the same for all, and the low one steps by bytes >> 4 from
// one MMA and stage to the next: one thread issues them all, another all copies,
// and with narrow tiles their instructions bound the kernel.  With descriptors
// put together for each MMA and addresses multiplied out for each stage,
// 64 x 4096 x 1024 in tiles of 16 rows takes 12.7 us, like this 8.9.
constexpr uint32_t DESC_HI = 1024u >> 4 | 1u << 14 | 2u << 29;

// (in a cluster an address carries the CTA's rank above the 18 bits of shared memory)
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, bool k_major)
{
    return (addr >> 4 & 0x3FFFu) | (k_major ? 1u : BOX_BYTES >> 4) << 16;
}

// from one MMA's 16 contraction elements to the next inside a stage
__device__ __forceinline__ uint32_t desc_step(bool k_major) { return (k_major ? UK * 2 : UK * 128) >> 4; }

__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, bool a_k_major, bool b_k_major, int M, int N)
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_k_major ? 0u : 1u) << 15) |
           ((b_k_major ? 0u : 1u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI)
        : "memory");
}

// a CTA pair's MMA, issued by its even CTA: A's 256 rows and B's N rows lie half
// in each CTA's shared memory, D's rows 0..127 in the even CTA's TMEM
__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI)
        : "memory");
}

template <Kind KIND>
struct Major {
    static constexpr bool a = KIND == kForward;      // A is K-major
    static constexpr bool b = KIND != kGradWeight;   // B is K-major
};

template <typename T, Kind KIND>
__host__ __device__ constexpr uint32_t idesc_of(int M, int N)
{
    return idesc_f16(std::is_same<T, __nv_bfloat16>::value, Major<KIND>::a, Major<KIND>::b, M, N);
}

// one stage of an operand tile, `width` of its M or N dimension from i0
template <bool K_MAJOR>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* tm, uint64_t* bar, int i0, int c0, int width)
{
    if (K_MAJOR) {
        tma_load_2d(dst, tm, bar, c0, i0);
    } else {
        for (int i = 0; i < width; i += 64) tma_load_2d(dst + (i / 64) * BOX_BYTES, tm, bar, i0 + i, c0);
    }
}

// ----------------------------------------------------------------------------
// Split kernel: a cluster of S CTAs computes one tile of 128 features x BN rows,
// each over its share of the contraction, and joins the S partial sums through
// distributed shared memory in rank order: no atomics and no second pass over
// memory, and results do not depend on timing.
//
//   warp 0     TMA producer (ring of `stages` boxes of A and B)
//   warp 1     TMEM allocation, tcgen05.mma issue
//   warps 0-7  epilogue, once the accumulator is complete
// ----------------------------------------------------------------------------
constexpr int SPLIT_THREADS = 256;
constexpr int JOIN = 4;          // rows that a warp joins at a time
constexpr int JOIN_LD = BM + 4;  // row distance of the partial sums: a lane quad's rows in different banks

struct SplitShape {
    int bn;      // rows t of a tile, a multiple of 16, <= 256
    int split;   // CTAs per tile
    int stages;
};

// bytes of a stage's `rows` rows of B; MN-major ones come in whole boxes of 64
template <Kind KIND>
__host__ __device__ constexpr int b_bytes(int rows)
{
    return Major<KIND>::b ? rows * BK * 2 : (rows + 63) / 64 * BOX_BYTES;
}
template <Kind KIND>
__host__ __device__ constexpr int stage_bytes(int bn) { return A_BYTES + b_bytes<KIND>(bn); }
__host__ __device__ constexpr uint32_t tmem_cols(int bn) { return bn <= 32 ? 32u : bn <= 64 ? 64u : bn <= 128 ? 128u : 256u; }

template <typename T, Kind KIND, bool READS, bool EXTRA>
__global__ void __launch_bounds__(SPLIT_THREADS, 2)
    split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const int kblocks,
                 const SplitShape sh, const __grid_constant__ Epilogue e)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int sbytes = stage_bytes<KIND>(sh.bn);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + sh.stages * sbytes);
    uint64_t* empty = full + MAX_STAGES;
    uint64_t* done = empty + MAX_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_id(), lane = lane_id();
    const int rank = sh.split > 1 ? (int)cluster_ctarank() : 0;
    const int tile = (int)(blockIdx.x / sh.split), mtiles = (e.m + BM - 1) / BM;
    const int f0 = tile % mtiles * BM, t0 = tile / mtiles * sh.bn;
    const int kb0 = (int)((int64_t)kblocks * rank / sh.split), kb1 = (int)((int64_t)kblocks * (rank + 1) / sh.split);
    const uint32_t cols = tmem_cols(sh.bn);
    if (threadIdx.x == 0) {
        for (int s = 0; s < sh.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) { tmem_alloc(tmem_slot, cols); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    start_of_inputs();

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0, started = 0;
            uint32_t ph = 0;
            uint8_t* sa = smem;
#pragma unroll 2
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&empty[stage], ph ^ 1u, abort_flag)) {
                    // let the copies already in flight land before the CTA exits
                    int never = 0;
                    for (int s = 0; s < min(started, sh.stages); ++s) {
                        const int i = started - 1 - s;
                        mbar_wait(&full[i % sh.stages], (uint32_t)(i / sh.stages) & 1u, &never, 20000000ull);
                    }
                    break;
                }
                mbar_arrive_expect_tx(&full[stage], sbytes);
                load_tile<Major<KIND>::a>(sa, &tmA, &full[stage], f0, kb * BK, BM);
                load_tile<Major<KIND>::b>(sa + A_BYTES, &tmB, &full[stage], t0, kb * BK, sh.bn);
                ++started;
                sa += sbytes;
                if (++stage == sh.stages) { stage = 0; ph ^= 1u; sa = smem; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (kb1 > kb0 && elect_one()) {
            const uint32_t idesc = idesc_of<T, KIND>(BM, sh.bn);
            const uint32_t a_first = desc_lo(smem_u32(smem), Major<KIND>::a), b_first = desc_lo(smem_u32(smem) + A_BYTES, Major<KIND>::b);
            int stage = 0;
            uint32_t ph = 0, at = 0;
#pragma unroll 2
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&full[stage], ph, abort_flag)) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < BK / UK; ++kk)
                    mma_f16(tmem, a_first + at + kk * desc_step(Major<KIND>::a), b_first + at + kk * desc_step(Major<KIND>::b), idesc,
                            kb > kb0 || kk ? 1u : 0u);
                mma_commit(&empty[stage]);
                at += (uint32_t)sbytes >> 4;
                if (++stage == sh.stages) { stage = 0; ph ^= 1u; at = 0; }
            }
            mma_commit(done);
        }
        __syncwarp();
    }
    // One CTA per tile: a warp takes its TMEM quarter's features and every other
    // 16 rows.  Several: the rows are dealt out to the warps of the cluster.
    const int rows = min(sh.bn, e.n - t0);  // rows of this tile that exist
    const bool joined = sh.split > 1;
    const int quarter = warp & 3, half = warp >> 2, fq = f0 + quarter * 32;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int f4 = f0 + lane * 4, mine = warp * sh.split + rank, deal = 8 * sh.split;
    Fetched<2> ahead;
    RowFetched ahead_rows[JOIN];
    float bias[4], sums[4] = {};
    if (!joined) {
        bias_of<T>(e, fq, bias);
        if (READS) fetch<T, KIND, 2>(e, fq, t0 + half * 16, ahead);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = e.bias && f4 + i < e.m ? to_f32(static_cast<const T*>(e.bias)[f4 + i]) : 0.0f;
        if (READS) {
#pragma unroll
            for (int u = 0; u < JOIN; ++u)
                if (mine + u * deal < rows) fetch_row<KIND>(e, f4, t0 + mine + u * deal, ahead_rows[u]);
        }
    }

    // every MMA of this CTA has completed (so every copy has landed and been read)
    bool ok = true;
    if (kb1 > kb0) ok = mbar_wait(done, 0, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();

    // the warps' memory: the ring's first, or behind the partial sums
    uint8_t* areas = smem + (joined ? sh.bn * JOIN_LD * 4 : 0);
    SettleList* list = &list_of(areas, warp);
    if (KIND == kForward && EXTRA) {
        if (lane == 0) list->count = 0;
        __syncwarp();
    }

    if (!joined) {
        const uint32_t stage = smem_u32(smem) + warp * kStageBytes;
        for (int c = half * 16; ok && c < rows; c += 32) {
            float v[16] = {};
            if (kblocks > 0) tmem_ld_frag<2>(tmem + lanes + c, v);
            finish<T, KIND, READS, EXTRA, 2>(e, fq, t0 + c, v, bias, ahead, {c + 32 < rows ? fq : -1, t0 + c + 32}, stage, sums, list);
        }
        if (KIND == kGradInput && EXTRA) put_sums(e, tile / mtiles * 2 + half, fq, sums);
    } else {
        // partial sums as [row][128 features] into the ring's shared memory
        float* part = reinterpret_cast<float*>(smem);
        const int at = (lane & 3) * 2 * JOIN_LD + (lane >> 2);  // of fragment 0
        for (int c = half * 16; c < rows; c += 32) {
            float v[16];
            tmem_ld_frag<2>(tmem + lanes + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                part[(c + (i >> 2 & 1) * 8 + (i & 1)) * JOIN_LD + quarter * 32 + (i >> 3) * 16 + (i >> 1 & 1) * 8 + at] = v[i];
        }
        cluster_sync();
        // a warp sums whole rows over the CTAs, 16 bytes a lane, in rank order
        const uint32_t here = smem_u32(part + lane * 4);
        for (int row = mine; row < rows; row += JOIN * deal) {
            float v[JOIN][4] = {};
            for (int r = 0; r < sh.split; ++r) {
                const uint32_t peer = map_to_rank(here, (uint32_t)r);
#pragma unroll
                for (int u = 0; u < JOIN; ++u)
                    if (row + u * deal < rows) {
                        const float4 w = ld_cluster_f32x4(peer + (uint32_t)((row + u * deal) * JOIN_LD * 4));
                        v[u][0] += w.x;
                        v[u][1] += w.y;
                        v[u][2] += w.z;
                        v[u][3] += w.w;
                    }
            }
#pragma unroll
            for (int u = 0; u < JOIN; ++u)
                if (ok && row + u * deal < rows) finish_row<T, KIND, READS, EXTRA>(e, f4, t0 + row + u * deal, v[u], bias, ahead_rows[u], sums, list);
            if (READS) {
#pragma unroll
                for (int u = 0; u < JOIN; ++u)
                    if (row + (JOIN + u) * deal < rows) fetch_row<KIND>(e, f4, t0 + row + (JOIN + u) * deal, ahead_rows[u]);
            }
        }
        if (KIND == kGradInput && EXTRA) {
            float* o = e.sums + ((int64_t)(tile / mtiles) * deal + mine) * e.m + f4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (f4 + i < e.m) o[i] = sums[i];
        }
        cluster_sync();  // no CTA leaves while another still reads its sums
    }
    if (KIND == kForward && EXTRA) {
        // every warp's codes and list are written; after a wait that ran out copies may still land on the lists
        if (__syncthreads_and(ok)) settle_all<T, SPLIT_THREADS / 32>(e, areas, threadIdx.x, [] { __syncthreads(); });
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, cols);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_status, CHPL_ERR_TIMEOUT);
}

// ----------------------------------------------------------------------------
// Pair kernel: persistent pairs of CTAs (tcgen05 cta_group::2), one tile of 256
// features x bn rows after another.  Each CTA stages 128 features of A and half
// of B's rows, so a stage feeds twice the multiply-adds per byte of shared
// memory that a lone CTA's would; the accumulator is double buffered in TMEM
// (2 x bn <= 512 columns), so the epilogue of one tile runs under the products
// of the next.
//
//   warp 0      TMA producer (both CTAs)
//   warp 1      TMEM allocation; tcgen05.mma issue (even CTA)
//   the others  epilogue (both CTAs)
// ----------------------------------------------------------------------------
// Sixteen epilogue warps with 16 rows each at a time: with a short contraction
// the epilogue's latencies bound the kernel, and four warps per scheduler hide
// them best (1024 x 1024 x 16384 with GELU and codes written 42 us; eight warps
// with 32 rows 47, with 16 rows 51; without either all three 28).
constexpr int PAIR_EPI_WARPS = 16;
constexpr int PAIR_NCB = 2;
constexpr int PAIR_THREADS = 64 + 32 * PAIR_EPI_WARPS;
constexpr int ROWS = 8 * PAIR_NCB;               // rows that an epilogue warp takes at a time
constexpr int ROUND = PAIR_EPI_WARPS / 4 * ROWS;  // rows that all of them do: a tile has as many at least
constexpr int PAIR_RING = 6 * (A_BYTES + 128 * BK * 2);  // bytes of the ring: six stages at 256 rows, more at fewer
constexpr int PAIR_SMEM = 1024 + PAIR_RING + PAIR_EPI_WARPS * kStageBytes + 512;

struct PairShape {
    int bn;              // rows t of a tile, a multiple of 32, 64 to 256
    int mtiles, ntiles;
    int group;           // feature tiles walked before the next row tile: see plan_for()
    int stages;          // of the ring
};

__device__ __forceinline__ void pair_tile(const PairShape& sh, int tile, int& mt, int& nt)
{
    const int per_group = sh.group * sh.ntiles;
    const int g = tile / per_group, first = g * sh.group;
    const int size = min(sh.group, sh.mtiles - first), local = tile - g * per_group;
    mt = first + local % size;
    nt = local / size;
}

template <bool K_MAJOR>
__device__ __forceinline__ void load_tile_pair(uint8_t* dst, const CUtensorMap* tm, uint32_t bar, int i0, int c0, int width)
{
    if (K_MAJOR) {
        tma_load_2d_pair(dst, tm, bar, c0, i0);
    } else {
        for (int i = 0; i < width; i += 64) tma_load_2d_pair(dst + (i / 64) * BOX_BYTES, tm, bar, i0 + i, c0);
    }
}

template <typename T, Kind KIND, bool READS, bool EXTRA>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const int kblocks,
                const PairShape sh, const __grid_constant__ Epilogue e)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int nstages = sh.stages, sbytes = A_BYTES + b_bytes<KIND>(sh.bn / 2);
    uint8_t* stages = smem + PAIR_RING;  // of the epilogue
    uint64_t* full = reinterpret_cast<uint64_t*>(stages + PAIR_EPI_WARPS * kStageBytes);
    uint64_t* empty = full + MAX_STAGES;
    uint64_t* acc_full = empty + MAX_STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster_ctarank();
    const int unit = (int)(blockIdx.x >> 1), nunits = (int)(gridDim.x >> 1);
    const int total = sh.mtiles * sh.ntiles;
    if (threadIdx.x == 0) {
        for (int s = 0; s < nstages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * PAIR_EPI_WARPS); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // barriers of the even CTA, where the MMAs are issued, as shared::cluster addresses
    const uint32_t lead_full = map_to_rank(smem_u32(full), 0), lead_acc_empty = map_to_rank(smem_u32(acc_empty), 0);
    const int half_rows = sh.bn / 2;
    start_of_inputs();

    if (warp == 0) {
        if (elect_one()) {
            const uint32_t bytes = 2u * (uint32_t)sbytes;  // both CTAs' copies
            int stage = 0, started = 0;
            uint32_t ph = 0;
            bool ok = true;
            uint8_t* sa = smem;
            for (int tile = unit; tile < total && ok; tile += nunits) {
                int mt, nt;
                pair_tile(sh, tile, mt, nt);
                const int f0 = mt * 2 * BM + (int)rank * BM, t0 = nt * sh.bn + (int)rank * half_rows;
#pragma unroll 2
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(&empty[stage], ph ^ 1u, abort_flag)) { ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
                    load_tile_pair<Major<KIND>::a>(sa, &tmA, lead_full + stage * 8, f0, kb * BK, BM);
                    load_tile_pair<Major<KIND>::b>(sa + A_BYTES, &tmB, lead_full + stage * 8, t0, kb * BK, half_rows);
                    ++started;
                    sa += sbytes;
                    if (++stage == nstages) { stage = 0; ph ^= 1u; sa = smem; }
                }
            }
            if (!ok) {  // let the copies already in flight land before the CTA exits
                const uint64_t t0 = globaltimer();
                while (globaltimer() - t0 < 1000000ull) {
                }
            } else {
                // every stage's last release (a commit of the even CTA's MMA thread) has landed here
                for (int s = 0; s < nstages; ++s) {
                    if (s >= nstages - started && !mbar_wait(&empty[stage], ph ^ 1u, abort_flag)) break;
                    if (++stage == nstages) { stage = 0; ph ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = idesc_of<T, KIND>(2 * BM, sh.bn);
            const uint32_t peer_empty = map_to_rank(smem_u32(empty), 1), peer_acc_full = map_to_rank(smem_u32(acc_full), 1);
            const uint32_t a_first = desc_lo(smem_u32(smem), Major<KIND>::a), b_first = desc_lo(smem_u32(smem) + A_BYTES, Major<KIND>::b);
            int stage = 0;
            uint32_t ph = 0, acc = 0, at = 0;
            bool ok = true;
            for (int tile = unit; tile < total && ok; tile += nunits) {
                const uint32_t buf = acc & 1u, aph = (acc >> 1) & 1u;
                if (!mbar_wait(&acc_empty[buf], aph ^ 1u, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d = tmem + buf * 256;
#pragma unroll 2
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(&full[stage], ph, abort_flag)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < BK / UK; ++kk)
                        mma_f16_pair(d, a_first + at + kk * desc_step(Major<KIND>::a), b_first + at + kk * desc_step(Major<KIND>::b), idesc,
                                     kb || kk ? 1u : 0u);
                    mma_commit_pair(smem_u32(&empty[stage]));
                    mma_commit_pair(peer_empty + stage * 8);
                    at += (uint32_t)sbytes >> 4;
                    if (++stage == nstages) { stage = 0; ph ^= 1u; at = 0; }
                }
                if (!ok) break;
                mma_commit_pair(smem_u32(&acc_full[buf]));
                mma_commit_pair(peer_acc_full + buf * 8);
                ++acc;
            }
            if (!ok) {  // the MMAs already issued complete before TMEM is released
                int never = 0;
                mma_commit_pair(smem_u32(drain));
                mbar_wait(drain, 0, &never, 20000000ull);
            } else {
                // both CTAs' epilogues have released both buffers (their arrivals have landed here)
                for (int b = 0; b < 2; ++b, ++acc)
                    if (!mbar_wait(&acc_empty[acc & 1u], ((acc >> 1) & 1u) ^ 1u, abort_flag)) break;
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        const int f_in = (int)rank * BM + quarter * 32;  // the warp's features within a tile
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t stage = smem_u32(stages) + (warp - 2) * kStageBytes;
        SettleList* list = &list_of(stages, warp - 2);
        if (KIND == kForward && EXTRA) {
            if (lane == 0) list->count = 0;
            __syncwarp();
        }
        uint32_t acc = 0;
        float sums[4] = {};
        int mt, nt;
        pair_tile(sh, unit, mt, nt);
        Fetched<PAIR_NCB> ahead;
        if (READS) fetch<T, KIND, PAIR_NCB>(e, mt * 2 * BM + f_in, nt * sh.bn + part * ROWS, ahead);
        for (int tile = unit; tile < total; tile += nunits, ++acc) {
            const int f = mt * 2 * BM + f_in, t0 = nt * sh.bn;
            const uint32_t buf = acc & 1u, aph = (acc >> 1) & 1u;
            float bias[4];
            bias_of<T>(e, f, bias);
            Next after = {-1, 0};  // the first rows of the next tile
            if (tile + nunits < total) {
                pair_tile(sh, tile + nunits, mt, nt);
                after = {mt * 2 * BM + f_in, nt * sh.bn + part * ROWS};
            }
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aph, abort_flag))) break;
            tc_fence_after();
            for (int c = part * ROWS; c < sh.bn; c += ROUND) {
                float v[ROWS];
                tmem_ld_frag<PAIR_NCB>(tmem + lanes + buf * 256 + c, v);
                const bool last = c + ROUND >= sh.bn;
                if (last) {  // this warp's last columns are in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_peer(lead_acc_empty + buf * 8);
                }
                finish<T, KIND, READS, EXTRA, PAIR_NCB>(e, f, t0 + c, v, bias, ahead, last ? after : Next{f, t0 + c + ROUND}, stage, sums,
                                                       list);
            }
            if (KIND == kGradInput && EXTRA) put_sums(e, t0 / sh.bn * (PAIR_EPI_WARPS / 4) + part, f, sums);
        }
        if (KIND == kForward && EXTRA) {
            const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(PAIR_EPI_WARPS * 32) : "memory"); };
            sync();  // every epilogue warp's codes and list are written
            settle_all<T, PAIR_EPI_WARPS>(e, stages, threadIdx.x - 64, sync);
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_status, CHPL_ERR_TIMEOUT);
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_fn()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Map of an operand with i (M or N dimension) < extent and c < k; box: 64
// contiguous elements by `box` of i (K-major) or by 64 of c (MN-major).
static int make_tmap(CUtensorMap* tm, const Operand& o, int64_t extent, int64_t k, int box)
{
    auto fn = encode_fn();
    if (!fn) { set_error("cuTensorMapEncodeTiled unavailable"); return CHPL_ERR_CUDA; }
    const int64_t inner = o.k_major ? k : extent, outer = o.k_major ? extent : k;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
    cuuint32_t boxes[2] = {64u, (cuuint32_t)(o.k_major ? box : BK)};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(o.p), dims, strides, boxes, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed (%d)", (int)r); return CHPL_ERR_CUDA; }
    return CHPL_OK;
}

int num_sms()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    return n;
}

// Which kernel, tile and split: the candidate of least estimated time.  The
// estimate, in us, is a start-up time and, for each wave of tiles that the SMs
// run, the staging of A and B per k-block and the epilogue, which a pair runs
// under the next tile; the join of a split comes on top.  A stage costs its
// bytes, 16 + bn / 8 KB for a lone CTA, at the rate of the SM (its ring of 216 KB
// over the latency of L2) or at that of L2 where all SMs stage; a pair's k-block
// also no less than its MMAs.  The constants are fitted to 3553 timings of 210
// products (profiles/linear_plan_timings.json; each kind, 1 to 8000 tokens, 64 to
// 16384 features): the choice is 2 % slower than the best candidate in the mean,
// a quarter at worst but for dW of some 30 tokens and fewer, one k-block a tile
// (1.4 to 1.6 times the best in three of them); one fixed tile was up to 5 times
// slower.  E.g. 512 x 4096 x 4096: a lone CTA's 128 rows 16.7 us, a pair's 128 rows
// 16.9, 256 rows 25.2, split in two 23.
//
// Large products run at the board's power limit, where traffic costs clock: a
// pair's tiles are walked in groups of features whose A, 32 MB of it, stays in
// L2 from one row tile to the next, 8 to 16 tiles.  Products of 1.1 TFLOP each,
// one after another: contraction 4096 in groups of 16 811 us, of 8 835, of 4 849;
// contraction 8192 876, 835, 861 (cuBLAS 780 to 815 for either).
struct Plan {
    bool pair;
    SplitShape split;
    PairShape tiles;
};

// CTAs of the split kernel that run at once, one or two to an SM: clusters of 4
// and 8 do not fill the GPU's processor clusters (132 and 120 of 148 SMs, 284 and
// 264 of 296 places, by the occupancy calculation for this GPU)
int slots(int split, int resident, int sms)
{
    const int lost = split <= 2 ? 0 : resident == 1 ? (split == 4 ? 16 : 28) : (split == 4 ? 12 : 32);
    return std::max(1, sms * resident - lost);
}

// the narrowest multiple of `step` rows that makes no more tiles of n rows than bn does
int fit_rows(int n, int bn, int step)
{
    const int tiles = (n + bn - 1) / bn;
    return (int)round_up((size_t)((n + tiles - 1) / tiles), (size_t)step);
}

SplitTime split_time(int stage_bytes, int bn, int64_t tiles, int split, int kblocks, int sms)
{
    const double ctas = (double)tiles * split, kbytes = stage_bytes / 1024.0, rest = 0.0078 * bn;
    // CTAs on an SM, two where one each does not hold them all: the SMs that hold two are the last to end
    const int resident = bn <= 64 && ctas > slots(split, 1, sms) ? 2 : 1, places = slots(split, resident, sms);
    const double stage = kbytes * std::max(0.0075, 0.0085 * std::min(1.0, ctas / places));
    return {2.26 + std::ceil(ctas / places) * (resident * ((kblocks + split - 1) / split * stage + rest) + 0.7) + (split > 1 ? 0.95 + 0.0147 * bn : 0.0),
            resident};
}

double pair_time(int stage_bytes, int bn, int64_t tiles, int kblocks, int sms)
{
    const double pairs = sms / 2, kbytes = stage_bytes / 1024.0, rest = 0.0072 * bn;
    const double stage = kbytes * std::max(0.0063, 0.0076 * std::min(1.0, tiles / pairs));
    const double products = kblocks * std::max(stage, 0.0013 * bn);
    return 3.1 + std::ceil(tiles / pairs) * (std::max(products, rest) + 0.42) + std::min(products, rest);
}

template <Kind KIND>
static Plan plan_for(int m, int n, int kblocks)
{
    const int sms = num_sms();
    Plan best;
    std::memset(&best, 0, sizeof(best));
    double least = 1e300;
    const int unit = Major<KIND>::b ? 16 : 64;  // rows: B's whole boxes where it is MN-major
    for (const int size : {16, 32, 48, 64, 96, 128, 192, 256}) {
        if (size % unit) continue;
        if (size >= 2 * n && least < 1e300) break;  // half the size holds every row
        const int bn = fit_rows(n, size, unit);
        const int64_t tiles = (int64_t)((m + BM - 1) / BM) * ((n + bn - 1) / bn);
        for (int split = 1; split <= 8 && (split == 1 || split <= kblocks); split *= 2) {
            const SplitTime e = split_time(stage_bytes<KIND>(bn), bn, tiles, split, kblocks, sms);
            if (e.us < least) {
                least = e.us;
                best.pair = false;
                best.split.bn = bn;
                best.split.split = split;
                best.split.stages = std::min(MAX_STAGES, (SMEM_LIMIT / e.resident - 2048) / stage_bytes<KIND>(bn));
            }
        }
    }
    // B's halves in whole boxes where it is MN-major
    const int step = Major<KIND>::b ? 32 : 128;
    for (int size = Major<KIND>::b ? ROUND : 128; size <= 256 && kblocks > 0 && n > size / 2; size += step) {
        const int bn = std::max(ROUND, fit_rows(n, size, step));
        const int64_t mt = (m + 2 * BM - 1) / (2 * BM), nt = (n + bn - 1) / bn;
        const double t = pair_time(A_BYTES + 2 * b_bytes<KIND>(bn / 2), bn, mt * nt, kblocks, sms);
        if (t < least && mt * nt < 0x7fffffff) {
            least = t;
            best.pair = true;
            best.tiles.bn = bn;
            best.tiles.mtiles = (int)mt;
            best.tiles.ntiles = (int)nt;
            best.tiles.group = std::max(8, std::min(16, 1024 / kblocks));
            best.tiles.stages = std::min(MAX_STAGES, PAIR_RING / (A_BYTES + b_bytes<KIND>(bn / 2)));
        }
    }
    return best;
}

template <typename T, Kind KIND, bool READS, bool EXTRA>
static int launch_split(cudaStream_t st, const Operand& a, const Operand& b, int64_t k, int kblocks, const Epilogue& e,
                        const SplitShape& s)
{
    const int64_t ctas = (int64_t)((e.m + BM - 1) / BM) * ((e.n + s.bn - 1) / s.bn) * s.split;
    if (ctas > 0x7fffffff) { set_error("linear: an output of %d x %d is more than one launch serves", e.n, e.m); return CHPL_ERR_UNSUPPORTED; }
    CUtensorMap tmA, tmB;
    std::memset(&tmA, 0, sizeof(tmA));
    std::memset(&tmB, 0, sizeof(tmB));
    if (kblocks > 0) {
        CHPL_TRY(make_tmap(&tmA, a, e.m, k, BM));
        CHPL_TRY(make_tmap(&tmB, b, e.n, k, s.bn));
    }
    static std::atomic<uint64_t> ready{0};
    CHPL_TRY(allow_smem(split_kernel<T, KIND, READS, EXTRA>, SMEM_LIMIT, ready));
    return launch_kernel(split_kernel<T, KIND, READS, EXTRA>, ctas, SPLIT_THREADS, 1024 + s.stages * stage_bytes<KIND>(s.bn) + 512, s.split, st,
                         tmA, tmB, kblocks, s, e);
}

template <typename T, Kind KIND, bool READS, bool EXTRA>
static int launch_pair(cudaStream_t st, const Operand& a, const Operand& b, int64_t k, int kblocks, const Epilogue& e,
                       const PairShape& s)
{
    CUtensorMap tmA, tmB;
    CHPL_TRY(make_tmap(&tmA, a, e.m, k, BM));
    CHPL_TRY(make_tmap(&tmB, b, e.n, k, s.bn / 2));
    static std::atomic<uint64_t> ready{0};
    CHPL_TRY(allow_smem(pair_kernel<T, KIND, READS, EXTRA>, PAIR_SMEM, ready));
    const int units = std::min(s.mtiles * s.ntiles, num_sms() / 2);
    return launch_kernel(pair_kernel<T, KIND, READS, EXTRA>, 2 * units, PAIR_THREADS, PAIR_SMEM, 2, st, tmA, tmB, kblocks, s, e);
}

template <typename T, Kind KIND, bool READS, bool EXTRA>
static int launch(cudaStream_t st, const Operand& a, const Operand& b, int64_t k, Epilogue& e)
{
    const int kblocks = (int)((k + BK - 1) / BK);
    const Plan p = plan_for<KIND>(e.m, e.n, kblocks);
    e.tie = tie_width(kblocks, p.pair ? 1 : p.split.split);
    return p.pair ? launch_pair<T, KIND, READS, EXTRA>(st, a, b, k, kblocks, e, p.tiles)
                  : launch_split<T, KIND, READS, EXTRA>(st, a, b, k, kblocks, e, p.split);
}

template <typename T, Kind KIND>
static int launch_kind(cudaStream_t st, const Operand& a, const Operand& b, int64_t k, Epilogue& e)
{
    if constexpr (KIND != kGradWeight)
        if (extra(KIND, e))
            return reads(KIND, e) ? launch<T, KIND, true, true>(st, a, b, k, e) : launch<T, KIND, false, true>(st, a, b, k, e);
    return reads(KIND, e) ? launch<T, KIND, true, false>(st, a, b, k, e) : launch<T, KIND, false, false>(st, a, b, k, e);
}

template <typename T>
static int launch_type(cudaStream_t st, Kind kind, const Operand& a, const Operand& b, int64_t k, Epilogue& e)
{
    if (kind == kForward) return launch_kind<T, kForward>(st, a, b, k, e);
    if (kind == kGradInput) return launch_kind<T, kGradInput>(st, a, b, k, e);
    return launch_kind<T, kGradWeight>(st, a, b, k, e);
}

int64_t sum_parts(int64_t m, int64_t n, int64_t k)
{
    if (m == 0 || n == 0) return 0;
    const Plan p = plan_for<kGradInput>((int)m, (int)n, (int)((k + BK - 1) / BK));
    if (p.pair) return (int64_t)p.tiles.ntiles * (PAIR_EPI_WARPS / 4);
    return (n + p.split.bn - 1) / p.split.bn * (p.split.split > 1 ? 8 * p.split.split : 2);
}

static int gemm_rows(cudaStream_t st, int type, Kind kind, const Operand& a, const Operand& b, int64_t k, Epilogue& e)
{
    const int elt = e.out_f32 ? 4 : 2;
    e.vec_out = aligned(e.out, e.ldo * elt, 16);
    e.vec_add = aligned(e.add, e.ldadd * elt, 16);
    e.vec_z = aligned(e.z, e.ldz * 2, 16);
    e.vec_codes = aligned(e.z8.codes, e.z8.ldc, 8);
    e.w = a.p;
    e.ldw = a.ld;
    e.x = b.p;
    e.ldx = b.ld;
    e.k = (int)k;
    return type == CHPL_TYPE_BF16 ? launch_type<__nv_bfloat16>(st, kind, a, b, k, e)
                                  : launch_type<__half>(st, kind, a, b, k, e);
}

// p, rows further
template <typename P>
static P* skip(P* p, int64_t rows, int64_t ld, int elt)
{
    return p ? reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(p) + (size_t)(rows * ld * elt)) : p;
}

int gemm(cudaStream_t st, int type, Kind kind, const Operand& a, const Operand& b, int64_t k, const Epilogue& e0)
{
    if (e0.m == 0 || e0.n == 0) return CHPL_OK;
    int64_t rows = e0.n;
    if (kind == kForward && extra(kind, e0)) {  // as many at a time as the warps' lists of codes to settle are made for
        const double outputs = settle_share(tie_width((int)((k + BK - 1) / BK), 1)) * PAIR_EPI_WARPS * num_sms();
        rows = std::min(rows, std::max<int64_t>(256, (int64_t)(outputs / e0.m)));
    }
    for (int64_t t = 0; t < e0.n; t += rows) {
        Epilogue e = e0;
        e.n = (int)std::min(rows, e0.n - t);
        e.out = skip(e.out, t, e.ldo, e.out_f32 ? 4 : 2);
        e.add = skip(e.add, t, e.ldadd, e.out_f32 ? 4 : 2);
        e.z = skip(e.z, t, e.ldz, 2);
        e.z8.codes = skip(e.z8.codes, t, e.z8.ldc, 1);
        e.z8.scales = skip(e.z8.scales, t, e.z8.lds, 1);
        Operand bt = b;
        if (t > 0) bt.p = skip(b.p, t, b.ld, 2);
        CHPL_TRY(gemm_rows(st, type, kind, a, bt, k, e));
    }
    return CHPL_OK;
}

// a wait on a phase that nothing completes, recorded as the kernels above record theirs
__global__ void diag_linear_wait_kernel(uint64_t limit_ns)
{
    __shared__ __align__(8) uint64_t bar;
    __shared__ int abort_flag;
    if (threadIdx.x != 0) return;
    mbar_init(&bar, 1);
    abort_flag = 0;
    fence_barrier_init();
    mbar_wait(&bar, 0, &abort_flag, limit_ns);
    if (*static_cast<volatile int*>(&abort_flag)) atomicExch(&g_status, CHPL_ERR_TIMEOUT);
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

extern "C" int chpl_diag_linear_wait(void* stream, uint64_t limit_ns)
{
    if (limit_ns == 0 || limit_ns > chpl::kWaitLimitNs) { chpl::set_error("limit_ns must be in (0, 2 s]"); return CHPL_ERR_INVALID; }
    chpl::linear::diag_linear_wait_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(limit_ns);
    CHPL_CUDA(cudaGetLastError());
    return CHPL_OK;
}

extern "C" int chpl_diag_linear_plan(int product, int64_t features, int64_t rows, int64_t contraction, int64_t plan[4])
{
    using namespace chpl::linear;
    const char* who = "diag_linear_plan";
    CHPL_TRY(check_size(who, "features", features));
    CHPL_TRY(check_size(who, "rows", rows));
    CHPL_TRY(check_size(who, "contraction", contraction));
    if (product < kForward || product > kGradWeight || !features || !rows || !plan) {
        chpl::set_error("%s: product 0, 1 or 2, features and rows above 0 and a plan are wanted", who);
        return CHPL_ERR_INVALID;
    }
    const int m = (int)features, n = (int)rows, kblocks = (int)((contraction + BK - 1) / BK);
    const Plan p = product == kForward     ? plan_for<kForward>(m, n, kblocks)
                   : product == kGradInput ? plan_for<kGradInput>(m, n, kblocks)
                                           : plan_for<kGradWeight>(m, n, kblocks);
    plan[0] = p.pair;
    plan[1] = p.pair ? p.tiles.bn : p.split.bn;
    plan[2] = p.pair ? 1 : p.split.split;
    plan[3] = p.pair ? (int64_t)p.tiles.mtiles * p.tiles.ntiles : (int64_t)((m + BM - 1) / BM) * ((n + p.split.bn - 1) / p.split.bn);
    return CHPL_OK;
}
