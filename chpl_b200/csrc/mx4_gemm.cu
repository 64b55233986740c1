// Products of 4-bit operands on the tensor cores: D[f][t] = sum over groups of 32
// c of 2^(sw + sx - 254) sum_c W(f, c) X(t, c), with the epilogue of the linear
// layers (linear_epilogue.cuh).
//
// tcgen05.mma kind::mxf4.block_scale multiplies E2M1 codes, two to a byte, 64 of
// the contraction at a time, and takes one E8M0 scale per row and 32 of them from
// TMEM.  Both operands are K-major; as in linear_gemm.cu the output's features
// lie along the TMEM lanes and its rows t along the columns, so a few tokens fill
// a narrow tile.  A stage holds 256 of the contraction: rows of 128 bytes of codes
// (TMA, 128-byte swizzle) and two blocks of scales, 128 rows x 4 groups in 512
// bytes each, which tcgen05.cp spreads over TMEM's lanes (32x128b.warpx4: lane l
// of every quarter gets bytes 16 l .. 16 l + 15, column i of them the scales of
// row 32 i + l).  The format keeps scales in that order in memory.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "linear_epilogue.cuh"
#include "mx4.h"

namespace chpl {
namespace linear {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
}
namespace mx4 {

using linear::Epilogue;
using linear::Fetched;
using linear::kForward;
using linear::kStageBytes;
using linear::Next;
using linear::RowFetched;

__device__ int g_status;  // sticky device-side error of this module

constexpr int BM = 128;                 // features of a tile (TMEM lanes)
constexpr int ROW_BYTES = kPiece / 2;   // of a stage's codes
constexpr int A_BYTES = BM * ROW_BYTES;
constexpr int SCALE_BYTES = 2 * kBlockBytes;  // a stage's scales of 128 rows
constexpr int STEPS = kPiece / 64;      // MMAs of a stage
constexpr int MAX_STAGES = 12;
constexpr int SMEM_LIMIT = 227 * 1024;

// ----------------------------------------------------------------------------
// tcgen05 kind::mxf4 with scales of 32
// ----------------------------------------------------------------------------
// A, B E2M1, scales E8M0, K-major, contraction 64; the scales of the first or the
// last two of four groups
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int groups)
{
    return ((uint32_t)groups << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) |
           ((uint32_t)groups << 29);
}

// K-major codes, 128-byte swizzle, 8-row groups 1024 bytes apart; the low word
// steps by 32 bytes from one MMA to the next
constexpr uint32_t DESC_HI = 1024u >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return (addr >> 4 & 0x3FFFu) | 1u << 16; }

// a block of scales: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart
constexpr uint32_t SCALE_HI = 128u >> 4 | 1u << 14;
__device__ __forceinline__ uint32_t scale_lo(uint32_t addr) { return addr >> 4 & 0x3FFFu; }

template <int GROUP>  // CTAs
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t lo)
{
    if (GROUP == 1)
        asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(lo), "n"(SCALE_HI) : "memory");
    else
        asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(lo), "n"(SCALE_HI) : "memory");
}

template <int GROUP>
__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t a_scale, uint32_t b_scale,
                                         uint32_t accumulate)
{
    if (GROUP == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "mov.b64 a, {%1, %5};\n\t"
            "mov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%6], [%7], p;\n\t}" ::"r"(d_tmem),
            "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI), "r"(a_scale), "r"(b_scale)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "mov.b64 a, {%1, %5};\n\t"
            "mov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%6], [%7], p;\n\t}" ::"r"(d_tmem),
            "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI), "r"(a_scale), "r"(b_scale)
            : "memory");
}

// One stage's products: its scales into TMEM (SCALE_COLS columns from `scales`),
// then four MMAs.  tcgen05.cp and tcgen05.mma of one thread execute in order, so
// the scales of a stage may replace those of two stages before.
constexpr int SCALE_COLS = 32;  // of a stage: A's two blocks in 0..7, B's 2 x up to 2 in 8..23
template <int GROUP>
__device__ __forceinline__ void stage_products(uint32_t d, uint32_t codes_lo, uint32_t b_off, uint32_t scales_lo, uint32_t scales, int b_blocks,
                                               uint32_t b_shift, uint32_t idesc, uint32_t idesc_high, bool first)
{
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        copy_scales<GROUP>(scales + 4 * q, scales_lo + (q * kBlockBytes >> 4));
        for (int b = 0; b < b_blocks; ++b)
            copy_scales<GROUP>(scales + 8 + 8 * q + 4 * b, scales_lo + (SCALE_BYTES * (1 + b) + q * kBlockBytes >> 4));
    }
#pragma unroll
    for (int kk = 0; kk < STEPS; ++kk)
        mma_mxf4<GROUP>(d, codes_lo + 2 * kk, codes_lo + b_off + 2 * kk, kk & 1 ? idesc_high : idesc, scales + 4 * (kk >> 1),
                        scales + 8 + 8 * (kk >> 1) + b_shift, first && kk == 0 ? 0u : 1u);
}

// ----------------------------------------------------------------------------
// Split kernel: a cluster of S CTAs computes one tile of 128 features x bn rows,
// each over its share of the contraction, and joins the partial sums through
// distributed shared memory in rank order, as the linear layers' does.
//
// CODES: X comes in 16 bits and every CTA codes its share of it itself, straight
// into the stages, four rows' 256 features a warp at a time: up to kCodedRows rows
// that needs no workspace and no launch before.  x 4096 x 16384, weights out of HBM,
// with GELU: one token 8.8 us, four 9.5, eight 10.8, coded first 10.2 to 10.4; x 4096
// x 28672 (two CTAs to an SM) 13.4, 13.2 and 13.8, coded first 14.8 to 15.0.  (Five to
// eight tokens, two units a stage, gain no GPU time on layers of up to 18944 features;
// the host launches once.)
//
//   warp 0     TMA producer          warp 1    TMEM allocation, tcgen05 issue
//   warps 2-7  CODES: X's codes and scales
//   warps 0-7  epilogue, once the accumulator is complete
// ----------------------------------------------------------------------------
constexpr int SPLIT_THREADS = 256;
constexpr int CODE_WARPS = SPLIT_THREADS / 32 - 2;
constexpr int CODE_ROWS = 4;     // that a warp codes at a time, a unit
constexpr int JOIN = 4;          // rows that a warp joins at a time
constexpr int JOIN_LD = BM + 4;  // row distance of the partial sums: a lane quad's rows in different banks

struct SplitShape {
    int bn;      // rows t of a tile: a multiple of 16, of 64 where there are several
    int split;   // CTAs per tile
    int stages;
};

// The units of a stage, and the warps that all units are dealt out to in order.  A
// warp waits until a stage's last use has been read by the parity of that use, which
// tells it from the use before, but not from the one before that.  With no more warps
// than one turn of the ring has units, a warp's units lie at most one turn apart.
// Stages are read in order, so what its last wait saw read covers the use before the
// last of the stage that it comes to: the parity can only mean the last one.  (Two
// CTAs to an SM have rings of five stages: five warps for up to four rows.)
__host__ __device__ constexpr int code_units(int rows) { return (rows + CODE_ROWS - 1) / CODE_ROWS; }
__host__ __device__ constexpr int code_warps(int stages, int rows)
{
    return CODE_WARPS < stages * code_units(rows) ? CODE_WARPS : stages * code_units(rows);
}

// blocks of scales that a tile's rows lie in: tiles start on multiples of 64
__host__ __device__ constexpr int row_blocks(int bn) { return bn <= 128 ? 1 : 2; }
__host__ __device__ constexpr int split_bytes(int bn) { return A_BYTES + bn * ROW_BYTES + (1 + row_blocks(bn)) * SCALE_BYTES; }
__host__ __device__ constexpr uint32_t tmem_cols(int bn)
{
    return bn + 2 * SCALE_COLS <= 128 ? 128u : bn + 2 * SCALE_COLS <= 256 ? 256u : 512u;
}

struct Maps {
    CUtensorMap w, x, sw, sx;  // codes and scales
};

template <typename T, bool READS, bool CODES>
__global__ void __launch_bounds__(SPLIT_THREADS, 2)
    split_kernel(const __grid_constant__ Maps tm, const RowsIn<T> x, const int k, const int kblocks, const SplitShape sh,
                 const __grid_constant__ Epilogue e)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int sbytes = split_bytes(sh.bn), b_blocks = row_blocks(sh.bn), codes = A_BYTES + sh.bn * ROW_BYTES;
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
        for (int s = 0; s < sh.stages; ++s) { mbar_init(&full[s], CODES ? 1 + code_units(e.n) : 1); mbar_init(&empty[s], 1); }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_barrier_init();
        if (kblocks > 0) {
            tma_prefetch_desc(&tm.w);
            tma_prefetch_desc(&tm.sw);
            if (!CODES) {
                tma_prefetch_desc(&tm.x);
                tma_prefetch_desc(&tm.sx);
            }
        }
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
                mbar_arrive_expect_tx(&full[stage], CODES ? A_BYTES + SCALE_BYTES : sbytes);
                tma_load_2d(sa, &tm.w, &full[stage], kb * ROW_BYTES, f0);
                tma_load_2d(sa + codes, &tm.sw, &full[stage], kb * (SCALE_BYTES / 4), f0 / kBlockRows);
                if (!CODES) {
                    tma_load_2d(sa + A_BYTES, &tm.x, &full[stage], kb * ROW_BYTES, t0);
                    tma_load_2d(sa + codes + SCALE_BYTES, &tm.sx, &full[stage], kb * (SCALE_BYTES / 4), t0 / kBlockRows);
                }
                ++started;
                sa += sbytes;
                if (++stage == sh.stages) { stage = 0; ph ^= 1u; sa = smem; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (kb1 > kb0 && elect_one()) {
            const uint32_t low = idesc_mxf4(BM, sh.bn, 0), high = idesc_mxf4(BM, sh.bn, 2);
            const uint32_t first = desc_lo(smem_u32(smem)), b_off = (uint32_t)A_BYTES >> 4, scales = tmem + (cols - 2 * SCALE_COLS);
            const uint32_t b_shift = (uint32_t)(t0 % kBlockRows) / 32;
            const uint32_t s_first = smem_u32(smem) + codes;
            int stage = 0;
            uint32_t ph = 0, at = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&full[stage], ph, abort_flag)) break;
                tc_fence_after();
                stage_products<1>(tmem, first + (at >> 4), b_off, scale_lo(s_first + at), scales + (kb & 1) * SCALE_COLS, b_blocks, b_shift, low,
                                  high, kb == kb0);
                mma_commit(&empty[stage]);
                at += (uint32_t)sbytes;
                if (++stage == sh.stages) { stage = 0; ph ^= 1u; at = 0; }
            }
            mma_commit(done);
        }
        __syncwarp();
    } else if (CODES && warp - 2 < code_warps(sh.stages, e.n)) {
        // units of CODE_ROWS rows in one stage, dealt out to the warps in order; the next
        // unit's rows are read while one is coded
        using Raw = typename RowsIn<T>::Raw;
        const int parts = code_units(e.n), units = (kb1 - kb0) * parts, coders = code_warps(sh.stages, e.n);
        Raw next[CODE_ROWS];
        const auto fetch = [&](int unit) {
            if (unit >= units) return;
            const int turn = unit / parts, row = (unit - turn * parts) * CODE_ROWS;
#pragma unroll
            for (int i = 0; i < CODE_ROWS; ++i)
                if (row + i < e.n) next[i] = x.raw(row + i, (kb0 + turn) * kPiece + lane * 8, k);
        };
        int unit = warp - 2;
        fetch(unit);
        for (; unit < units; unit += coders) {
            const int turn = unit / parts, row = (unit - turn * parts) * CODE_ROWS, stage = turn % sh.stages;
            Raw raw[CODE_ROWS];
            uint32_t w[CODE_ROWS], s[CODE_ROWS];
#pragma unroll
            for (int i = 0; i < CODE_ROWS; ++i) raw[i] = next[i];
            fetch(unit + coders);
#pragma unroll
            for (int i = 0; i < CODE_ROWS; ++i) {
                s[i] = x.top(raw[i]);
                s[i] = max(s[i], __shfl_xor_sync(0xffffffffu, s[i], 1));
                s[i] = scale_of(max(s[i], __shfl_xor_sync(0xffffffffu, s[i], 2)));
                float v[8];
                x.value(raw[i], v);
                w[i] = codes8(v, inv_step(s[i]));
                if (s[i] == kBadScale) w[i] = 0;
            }
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], (uint32_t)(turn / sh.stages & 1) ^ 1u, abort_flag))) break;
            const uint32_t at = smem_u32(smem) + stage * sbytes;
#pragma unroll
            for (int i = 0; i < CODE_ROWS; ++i) {
                if (row + i >= e.n) break;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + A_BYTES + (row + i) * ROW_BYTES + (((lane >> 2) ^ (row + i & 7)) << 4) + (lane & 3) * 4),
                             "r"(w[i])
                             : "memory");
                if ((lane & 3) == 0)
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(at + codes + SCALE_BYTES + (lane >> 4) * kBlockBytes + (row + i) * 16 + (lane >> 2 & 3)),
                                 "r"(s[i])
                                 : "memory");
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
        }
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
        linear::bias_of<T>(e, fq, bias);
        if (READS) linear::fetch<T, kForward, 2>(e, fq, t0 + half * 16, ahead);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = e.bias && f4 + i < e.m ? to_f32(static_cast<const T*>(e.bias)[f4 + i]) : 0.0f;
        if (READS) {
#pragma unroll
            for (int u = 0; u < JOIN; ++u)
                if (mine + u * deal < rows) linear::fetch_row<kForward>(e, f4, t0 + mine + u * deal, ahead_rows[u]);
        }
    }

    // every MMA of this CTA has completed (so every copy has landed and been read)
    bool ok = true;
    if (kb1 > kb0) ok = mbar_wait(done, 0, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (!joined) {
        const uint32_t stage = smem_u32(smem) + warp * kStageBytes;
        for (int c = half * 16; ok && c < rows; c += 32) {
            float v[16] = {};
            if (kblocks > 0) linear::tmem_ld_frag<2>(tmem + lanes + c, v);
            linear::finish<T, kForward, READS, false, 2>(e, fq, t0 + c, v, bias, ahead, {c + 32 < rows ? fq : -1, t0 + c + 32}, stage, sums,
                                                         nullptr);
        }
    } else {
        // partial sums as [row][128 features] into the ring's shared memory
        float* part = reinterpret_cast<float*>(smem);
        const int at = (lane & 3) * 2 * JOIN_LD + (lane >> 2);  // of fragment 0
        for (int c = half * 16; c < rows; c += 32) {
            float v[16];
            linear::tmem_ld_frag<2>(tmem + lanes + c, v);
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
                        const float4 w = linear::ld_cluster_f32x4(peer + (uint32_t)((row + u * deal) * JOIN_LD * 4));
                        v[u][0] += w.x;
                        v[u][1] += w.y;
                        v[u][2] += w.z;
                        v[u][3] += w.w;
                    }
            }
#pragma unroll
            for (int u = 0; u < JOIN; ++u)
                if (ok && row + u * deal < rows)
                    linear::finish_row<T, kForward, READS, false>(e, f4, t0 + row + u * deal, v[u], bias, ahead_rows[u], sums, nullptr);
            if (READS) {
#pragma unroll
                for (int u = 0; u < JOIN; ++u)
                    if (row + (JOIN + u) * deal < rows) linear::fetch_row<kForward>(e, f4, t0 + row + (JOIN + u) * deal, ahead_rows[u]);
            }
        }
        cluster_sync();  // no CTA leaves while another still reads its sums
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
// Pair kernel: persistent pairs of CTAs (cta_group::2), one tile of 256 features
// x bn rows after another.  Each CTA stages its 128 features of W with their
// scales, half of X's rows, and the scales of all of X's rows, which both CTAs'
// tensor cores need.
//
// At this rate of products the copies out of L2 bound large tiles, some 11 TB/s
// over all SMs, so tiles are as wide as an MMA: 256 rows.  Two accumulators of 256
// columns and the scales do not fit in TMEM's 512 columns; the second one starts
// at column 192, and a tile's epilogue takes the 64 columns that both share first.
// The next tile's products start when those have been read (32 arrivals), the
// other columns are read under them.  A warp that has arrived for a tile has read
// all it reads of the tile before, whose other columns the next one overwrites.
// 8192 x 4096 x 16384 with GELU: 220 us, 5.0 PFLOP/s (243 with tiles of 192 rows and
// accumulators apart); without copies into the stages 174, without outputs 167.
//
//   warp 0      TMA producer (both CTAs)
//   warp 1      TMEM allocation; tcgen05 issue (even CTA)
//   the others  epilogue (both CTAs)
// ----------------------------------------------------------------------------
constexpr int PAIR_EPI_WARPS = 16;
constexpr int PAIR_NCB = 2;
constexpr int PAIR_THREADS = 64 + 32 * PAIR_EPI_WARPS;
constexpr int ROWS = 8 * PAIR_NCB;                // rows that an epilogue warp takes at a time
constexpr int ROUND = PAIR_EPI_WARPS / 4 * ROWS;  // rows that all of them do
constexpr int PAIR_MAX_BN = 256;
constexpr int ACC_STEP = 192;                     // columns from one accumulator to the next
constexpr int SCALES_AT = 512 - 2 * SCALE_COLS;   // the second one ends here
static_assert(ACC_STEP + PAIR_MAX_BN == SCALES_AT && PAIR_MAX_BN - ACC_STEP == ROUND, "TMEM");
constexpr int PAIR_RING = SMEM_LIMIT - 1024 - PAIR_EPI_WARPS * kStageBytes - 512;

struct PairShape {
    int bn;              // rows t of a tile: 64, 128, 192 or 256
    int mtiles, ntiles;
    int group;           // feature tiles walked before the next row tile
    int stages;
};

__host__ __device__ constexpr int pair_bytes(int bn) { return A_BYTES + bn / 2 * ROW_BYTES + (1 + row_blocks(bn)) * SCALE_BYTES; }

__device__ __forceinline__ void pair_tile(const PairShape& sh, int tile, int& mt, int& nt)
{
    const int per_group = sh.group * sh.ntiles;
    const int g = tile / per_group, first = g * sh.group;
    const int size = min(sh.group, sh.mtiles - first), local = tile - g * per_group;
    mt = first + local % size;
    nt = local / size;
}

template <typename T, bool READS>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ Maps tm, const int kblocks, const PairShape sh, const __grid_constant__ Epilogue e)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int nstages = sh.stages, sbytes = pair_bytes(sh.bn), half_rows = sh.bn / 2, b_blocks = row_blocks(sh.bn);
    const int codes = A_BYTES + half_rows * ROW_BYTES;
    uint8_t* stages = smem + nstages * sbytes;  // of the epilogue
    uint64_t* full = reinterpret_cast<uint64_t*>(stages + PAIR_EPI_WARPS * kStageBytes);
    uint64_t* empty = full + MAX_STAGES;
    uint64_t* acc_full = empty + MAX_STAGES;
    uint64_t* acc_read = acc_full + 2;  // what the next accumulator overwrites
    uint64_t* drain = acc_read + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster_ctarank();
    const int unit = (int)(blockIdx.x >> 1), nunits = (int)(gridDim.x >> 1);
    const int total = sh.mtiles * sh.ntiles;
    if (threadIdx.x == 0) {
        for (int s = 0; s < nstages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) mbar_init(&acc_full[b], 1);
        mbar_init(acc_read, 2 * PAIR_EPI_WARPS);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm.w);
        tma_prefetch_desc(&tm.x);
        tma_prefetch_desc(&tm.sw);
        tma_prefetch_desc(&tm.sx);
    }
    if (warp == 1) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // barriers of the even CTA, where the MMAs are issued, as shared::cluster addresses
    const uint32_t lead_full = map_to_rank(smem_u32(full), 0), lead_acc_read = map_to_rank(smem_u32(acc_read), 0);
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
                const int f0 = mt * 2 * BM + (int)rank * BM, t0 = nt * sh.bn;
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(&empty[stage], ph ^ 1u, abort_flag)) { ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
                    const uint32_t bar = lead_full + stage * 8;
                    tma_load_2d_pair(sa, &tm.w, bar, kb * ROW_BYTES, f0);
                    tma_load_2d_pair(sa + A_BYTES, &tm.x, bar, kb * ROW_BYTES, t0 + (int)rank * half_rows);
                    tma_load_2d_pair(sa + codes, &tm.sw, bar, kb * (SCALE_BYTES / 4), f0 / kBlockRows);
                    tma_load_2d_pair(sa + codes + SCALE_BYTES, &tm.sx, bar, kb * (SCALE_BYTES / 4), t0 / kBlockRows);
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
            const uint32_t low = idesc_mxf4(2 * BM, sh.bn, 0), high = idesc_mxf4(2 * BM, sh.bn, 2);
            const uint32_t peer_empty = map_to_rank(smem_u32(empty), 1), peer_acc_full = map_to_rank(smem_u32(acc_full), 1);
            const uint32_t first = desc_lo(smem_u32(smem)), b_off = (uint32_t)A_BYTES >> 4, scales = tmem + SCALES_AT;
            const uint32_t s_first = smem_u32(smem) + codes;
            int stage = 0;
            uint32_t ph = 0, acc = 0, at = 0, turn = 0;
            bool ok = true;
            for (int tile = unit; tile < total && ok; tile += nunits) {
                int mt, nt;
                pair_tile(sh, tile, mt, nt);
                const uint32_t b_shift = (uint32_t)(nt * sh.bn % kBlockRows) / 32;
                const uint32_t buf = acc & 1u;
                if (acc > 0 && !mbar_wait(acc_read, (acc - 1) & 1u, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d = tmem + buf * ACC_STEP;
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(&full[stage], ph, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    stage_products<2>(d, first + (at >> 4), b_off, scale_lo(s_first + at), scales + turn * SCALE_COLS, b_blocks, b_shift, low, high,
                                      kb == 0);
                    mma_commit_pair(smem_u32(&empty[stage]));
                    mma_commit_pair(peer_empty + stage * 8);
                    at += (uint32_t)sbytes;
                    turn ^= 1u;
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
                // both CTAs' epilogues have arrived for the last tile (the arrivals have landed here)
                if (acc > 0) mbar_wait(acc_read, (acc - 1) & 1u, abort_flag);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        const int f_in = (int)rank * BM + quarter * 32;  // the warp's features within a tile
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t stage = smem_u32(stages) + (warp - 2) * kStageBytes;
        uint32_t acc = 0;
        float sums[4] = {};
        int mt, nt;
        pair_tile(sh, unit, mt, nt);
        // A tile's rounds of 64 rows, the one that lies in both accumulators first: the
        // first accumulator's from column 192 (if it has them), the second one's from 0.
        const int rounds = sh.bn / ROUND;
        const auto rows_of = [&](uint32_t buf, int r) {
            const int first = buf == 0 && sh.bn > ACC_STEP ? ACC_STEP / ROUND : 0;
            return (r + first < rounds ? r + first : r + first - rounds) * ROUND + part * ROWS;
        };
        Fetched<PAIR_NCB> ahead;
        if (READS) linear::fetch<T, kForward, PAIR_NCB>(e, mt * 2 * BM + f_in, nt * sh.bn + rows_of(0, 0), ahead);
        for (int tile = unit; tile < total; tile += nunits, ++acc) {
            const int f = mt * 2 * BM + f_in, t0 = nt * sh.bn;
            const uint32_t buf = acc & 1u, aph = (acc >> 1) & 1u;
            float bias[4];
            linear::bias_of<T>(e, f, bias);
            Next after = {-1, 0};  // the first rows of the next tile
            if (tile + nunits < total) {
                pair_tile(sh, tile + nunits, mt, nt);
                after = {mt * 2 * BM + f_in, nt * sh.bn + rows_of(buf ^ 1u, 0)};
            }
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aph, abort_flag))) break;
            tc_fence_after();
            for (int r = 0; r < rounds; ++r) {
                const int c = rows_of(buf, r);
                float v[ROWS];
                linear::tmem_ld_frag<PAIR_NCB>(tmem + lanes + buf * ACC_STEP + c, v);
                if (r == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) linear::mbar_arrive_peer(lead_acc_read);
                }
                linear::finish<T, kForward, READS, false, PAIR_NCB>(e, f, t0 + c, v, bias, ahead, r + 1 == rounds ? after : Next{f, t0 + rows_of(buf, r + 1)},
                                                                    stage, sums, nullptr);
            }
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
// rows of `bytes` bytes, `ld` apart, in boxes of `box` rows
static int make_tmap(CUtensorMap* tm, CUtensorMapDataType type, int elt, const void* p, int64_t width, int64_t rows, int64_t ld_bytes, int box_width,
                     int box, CUtensorMapSwizzle swizzle)
{
    auto fn = linear::encode_fn();
    if (!fn) { set_error("cuTensorMapEncodeTiled unavailable"); return CHPL_ERR_CUDA; }
    cuuint64_t dims[2] = {(cuuint64_t)(width / elt), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld_bytes};
    cuuint32_t boxes[2] = {(cuuint32_t)(box_width / elt), (cuuint32_t)box};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(tm, type, 2, const_cast<void*>(p), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed (%d)", (int)r); return CHPL_ERR_CUDA; }
    return CHPL_OK;
}

// x.codes NULL: X has no maps
static int make_maps(Maps* tm, const chpl_mx4& w, const chpl_mx4& x, int m, int n, int64_t k, int x_box, int x_blocks)
{
    const int64_t width = code_bytes(k), scales = blocks_of(k) * kBlockBytes;
    // one row has no distance
    const int64_t ldw = m > 1 ? w.ldc : width, ldx = n > 1 ? x.ldc : width;
    CHPL_TRY(make_tmap(&tm->w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.codes, width, m, ldw, ROW_BYTES, BM, CU_TENSOR_MAP_SWIZZLE_128B));
    CHPL_TRY(make_tmap(&tm->sw, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, w.scales, scales, (m + kBlockRows - 1) / kBlockRows, scales, SCALE_BYTES, 1,
                       CU_TENSOR_MAP_SWIZZLE_NONE));
    if (!x.codes) return CHPL_OK;
    CHPL_TRY(make_tmap(&tm->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x.codes, width, n, ldx, ROW_BYTES, x_box, CU_TENSOR_MAP_SWIZZLE_128B));
    return make_tmap(&tm->sx, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, x.scales, scales, (n + kBlockRows - 1) / kBlockRows, scales, SCALE_BYTES, x_blocks,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Which kernel, tile and split: the candidate of least estimated time, the linear
// layers' estimate (linear_gemm.cu) with this module's stages, which are as many
// bytes.  Of 1302 timings of 120 products (profiles/mx4_plan_timings.json; 1 to 8192
// tokens, 64 to 16384 features) the choice is 1 % slower than the best candidate in
// the mean, 19 % at worst; constants fitted to these timings chose no better.
struct Plan {
    bool pair;
    SplitShape split;
    PairShape tiles;
};

static Plan plan_for(int m, int n, int kblocks)
{
    const int sms = linear::num_sms();
    Plan best;
    std::memset(&best, 0, sizeof(best));
    double least = 1e300;
    for (const int size : {16, 32, 48, 64, 96, 128, 192, 256}) {
        if (size >= 2 * n && least < 1e300) break;  // half the size holds every row
        if (n > size && size % 64) continue;        // several tiles start on multiples of 64
        const int bn = linear::fit_rows(n, size, n > size ? 64 : 16);
        const int64_t tiles = (int64_t)((m + BM - 1) / BM) * ((n + bn - 1) / bn);
        for (int split = 1; split <= 8 && (split == 1 || split <= kblocks); split *= 2) {
            const linear::SplitTime e = linear::split_time(split_bytes(bn), bn, tiles, split, kblocks, sms);
            if (e.us < least) {
                least = e.us;
                best.pair = false;
                best.split.bn = bn;
                best.split.split = split;
                best.split.stages = std::min(MAX_STAGES, (SMEM_LIMIT / e.resident - 2048) / split_bytes(bn));
            }
        }
    }
    for (int bn = 64; bn <= PAIR_MAX_BN && kblocks > 0 && n > bn / 2; bn += 64) {
        const int64_t mt = (m + 2 * BM - 1) / (2 * BM), nt = (n + bn - 1) / bn;
        const double t = linear::pair_time(A_BYTES + bn * ROW_BYTES + 3 * SCALE_BYTES, bn, mt * nt, kblocks, sms);
        if (t < least && mt * nt < 0x7fffffff) {
            least = t;
            best.pair = true;
            best.tiles.bn = bn;
            best.tiles.mtiles = (int)mt;
            best.tiles.ntiles = (int)nt;
            best.tiles.group = 16;
            best.tiles.stages = std::min(MAX_STAGES, PAIR_RING / pair_bytes(bn));
        }
    }
    return best;
}

template <typename T, bool READS, bool CODES>
static int launch_split(cudaStream_t st, const Maps& tm, const RowsIn<T>& x, int64_t k, int kblocks, const SplitShape& s, const Epilogue& e)
{
    const int64_t ctas = (int64_t)((e.m + BM - 1) / BM) * ((e.n + s.bn - 1) / s.bn) * s.split;
    if (ctas > 0x7fffffff) { set_error("mx4_linear: an output of %d x %d is more than one launch serves", e.n, e.m); return CHPL_ERR_UNSUPPORTED; }
    static std::atomic<uint64_t> ready{0};
    CHPL_TRY(allow_smem(split_kernel<T, READS, CODES>, SMEM_LIMIT, ready));
    return launch_kernel(split_kernel<T, READS, CODES>, ctas, SPLIT_THREADS, 1024 + s.stages * split_bytes(s.bn) + 512, s.split, st, tm, x, (int)k,
                         kblocks, s, e);
}

template <typename T, bool READS>
static int launch(cudaStream_t st, const chpl_mx4& w, const chpl_mx4& x, const void* x16, int64_t ldx, int64_t k, const Epilogue& e)
{
    const int kblocks = (int)((k + kPiece - 1) / kPiece);
    const Plan p = plan_for(e.m, e.n, kblocks);
    Maps tm;
    std::memset(&tm, 0, sizeof(tm));
    if (p.pair) {
        const PairShape& s = p.tiles;
        CHPL_TRY(make_maps(&tm, w, x, e.m, e.n, k, s.bn / 2, row_blocks(s.bn)));
        static std::atomic<uint64_t> ready{0};
        CHPL_TRY(allow_smem(pair_kernel<T, READS>, SMEM_LIMIT, ready));
        const int units = std::min(s.mtiles * s.ntiles, linear::num_sms() / 2);
        return launch_kernel(pair_kernel<T, READS>, 2 * units, PAIR_THREADS, 1024 + s.stages * pair_bytes(s.bn) + PAIR_EPI_WARPS * kStageBytes + 512, 2,
                             st, tm, kblocks, s, e);
    }
    if (kblocks > 0) CHPL_TRY(make_maps(&tm, w, x, e.m, e.n, k, p.split.bn, row_blocks(p.split.bn)));
    const RowsIn<T> rows = rows_in<T>(x16, ldx);
    return x16 ? launch_split<T, READS, true>(st, tm, rows, k, kblocks, p.split, e) : launch_split<T, READS, false>(st, tm, rows, k, kblocks, p.split, e);
}

int gemm(cudaStream_t st, int type, const chpl_mx4& w, const chpl_mx4& x, const void* x16, int64_t ldx, int64_t k, const Epilogue& e0)
{
    Epilogue e = e0;
    e.vec_out = aligned(e.out, e.ldo * 2, 16);
    e.vec_add = aligned(e.add, e.ldadd * 2, 16);
    if (type == CHPL_TYPE_BF16) return e.add ? launch<__nv_bfloat16, true>(st, w, x, x16, ldx, k, e) : launch<__nv_bfloat16, false>(st, w, x, x16, ldx, k, e);
    return e.add ? launch<__half, true>(st, w, x, x16, ldx, k, e) : launch<__half, false>(st, w, x, x16, ldx, k, e);
}

int read_clear_status(int* st)
{
    int v = 0, z = 0;
    CHPL_CUDA(cudaMemcpyFromSymbol(&v, g_status, sizeof(int)));
    CHPL_CUDA(cudaMemcpyToSymbol(g_status, &z, sizeof(int)));
    *st = v;
    return CHPL_OK;
}

}  // namespace mx4
}  // namespace chpl

extern "C" int chpl_diag_mx4_ring(int64_t features, int64_t rows, int64_t contraction, int64_t ring[3])
{
    using namespace chpl::mx4;
    const char* who = "diag_mx4_ring";
    CHPL_TRY(chpl::linear::check_size(who, "features", features));
    CHPL_TRY(chpl::linear::check_size(who, "rows", rows));
    CHPL_TRY(chpl::linear::check_size(who, "contraction", contraction));
    if (!ring || !features || !rows) { chpl::set_error("%s: nothing to plan", who); return CHPL_ERR_INVALID; }
    const Plan p = plan_for((int)features, (int)rows, (int)((contraction + kPiece - 1) / kPiece));
    const bool coded = rows <= kCodedRows;
    ring[0] = p.pair ? p.tiles.stages : p.split.stages;
    ring[1] = coded ? code_units((int)rows) : 0;
    ring[2] = coded ? code_warps(p.split.stages, (int)rows) : 0;
    return CHPL_OK;
}

extern "C" int chpl_diag_mx4_plan(int64_t features, int64_t rows, int64_t contraction, int64_t plan[3])
{
    using namespace chpl::mx4;
    const char* who = "diag_mx4_plan";
    CHPL_TRY(chpl::linear::check_size(who, "features", features));
    CHPL_TRY(chpl::linear::check_size(who, "rows", rows));
    CHPL_TRY(chpl::linear::check_size(who, "contraction", contraction));
    if (!plan || !features || !rows) { chpl::set_error("%s: nothing to plan", who); return CHPL_ERR_INVALID; }
    const Plan p = plan_for((int)features, (int)rows, (int)((contraction + kPiece - 1) / kPiece));
    plan[0] = p.pair;
    plan[1] = p.pair ? p.tiles.bn : p.split.bn;
    plan[2] = p.pair ? 1 : p.split.split;
    return CHPL_OK;
}
