// Block-scaled e4m3 GEMM for sm_100a on the 5th-generation tensor cores:
//   D[m,n] = sum over 128-wide blocks b of K of
//            a_scale[m,b] * b_scale[n/128,b] * sum_{k in b} A[m,k] * B_T[n,k]
// dense (M, N, K) and grouped by device-side row offsets (expert e owns rows
// [offsets[e], offsets[e+1]) of A and D and its own N rows of B_T; any alignment).
//
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4, f32 accumulation in TMEM), one
// accumulator for each block of K; the scales are f32 and differ from row to row, so the outer sum
// runs in registers: the epilogue warps fetch each block's accumulator from TMEM, multiply it by the
// row's scale times the weight block's and add it to the tile's f32 sums.  128 rows are the 128 TMEM
// lanes, so a thread has one row: one scale for a block of K, and its columns lie in one weight block.
// The two scales are multiplied first, in f32, one product a block: products below 2^-126 lose bits (2^-125 of a block's
// result at most) and those of 2^128 are infinite.  Looking out for them costs every call more than it gives: a vote a
// block and a branch 239 us at 8192 x 8192 x 4096 where 215 were measured without, a look by the warp that copies the scales
// 229, sums kept at 2^24 times their value 217 (and those overflow sooner).
//
// What bounds it at large sizes: a CTA's 128 x 256 x 128 block takes 512 clocks of MMA, 512 of operands
// from L2 (64 bytes a clock), and the drain of its accumulators 286 clocks of each SM sub-partition's
// TMEM port and FMA pipe.  The three overlap, but the way MMA -> commit -> epilogue -> release -> MMA
// is long, TMEM holds two blocks, and the instructions that issue a block's MMAs take nearly as long as the
// MMAs: a block takes 690 clocks (630 with an epilogue that only hands accumulators back), plus 3000 a tile
// for its store and the restart (1400 of them go without the writes themselves).  8192 x 8192 x 4096: 224 us,
// 2450 TFLOP/s back to back; 2110 when run for seconds, under the power cap.
// What brought it there (8192 x 8192 x 4096): pairs of CTAs with four accumulators of 128 columns instead of
// two of 256, so that a half is released while the other runs; MMAs issued from uniform registers by an
// elected lane (from a lane's own they issue at 60 clocks each); the next barriers looked at under the
// current work, in the issuing warp and in the epilogue; scales copied into shared memory a group of
// blocks ahead (read from global memory by the epilogue they cost 700 clocks a block); fewer instructions
// between one half's MMAs and the next, and accumulators handed back after two batches of loads: 345 -> 224 us.
// Two issuing warps, 16 epilogue warps with 64 columns each, warps that take 64 columns of both halves, and
// accumulators of 256 columns measured slower.
//
// Structure as the bf16 GEMM's (gemm_sm100.cu): persistent, one warp = TMA producer, one = MMA issuer and
// TMEM owner, one copies scales, the epilogue's warps two for each quarter of the lanes, each with half of
// the columns.  Bounded waits throughout.
#include "common.cuh"
#include "ptx.cuh"
#include "fmha_math.cuh"

#include <cuda_bf16.h>

#include <atomic>

namespace pb200 {
namespace {

using namespace ptx;

constexpr int BM = 128;
constexpr int BK = 128;                      // one scale block of K = one 128-byte swizzle row of e4m3
constexpr int kSmallRows = 32;               // row box of A for tiles with few rows, and all of A in the few-rows form
constexpr int kRingBytes = 200 * 1024;       // operand ring and store boxes
constexpr int kBoxBytes = 32 * 128;          // a warp's store box: 32 rows of 128 bytes
constexpr int kBoxes = 2;                    // of them in flight for each epilogue warp
constexpr int kLaunchThreads = 384;          // 128-row forms: 4 warps of control, 8 of epilogue
constexpr int kFewThreads = 256;             // 32-row forms: 3 warps of control, 2 of epilogue (both on lanes 0-31), 3 that only
                                             // help to add partial tiles (registers are handed out for 8 warps anyway)
constexpr int kAccCols = 128;                // TMEM columns of an accumulator
constexpr int kMaxExperts = 1024;
constexpr int kTableBytes = 2 * (kMaxExperts + 1) * 4 + 120;      // sanitised offsets and tile prefix, padded to 128
constexpr int kBarBytes = 1024;
constexpr int kGroup = 8;                    // scale blocks whose scales are fetched together (one 32-byte sector of a row)
constexpr int kScaleWords = kGroup * BM + 2 * kGroup;             // of a group: 128 rows', two column blocks'
constexpr int kScaleBytes = (2 * kScaleWords * 4 + 127) / 128 * 128;
constexpr int kSmemTotal = 1024 + kRingBytes + kTableBytes + kScaleBytes + kBarBytes;
constexpr int kPartPitch = 128 + 4;          // f32 row pitch of a split's partial tile: rows on distinct banks
static_assert(kSmemTotal <= 227 * 1024, "shared memory");
constexpr int kMaxSplit = 8;
// Registers of the 256-column form, whose epilogue threads hold 128 sums: the launch has 384 x 168;
// the control warpgroup gives up 128 x 112 of them and the two epilogue warpgroups take 256 x 56 (with 16 a
// thread more for these and as many less for the control warps, the control warps spill; as it is, ptxas reports 12 bytes of
// spill stores for bf16 results and none for f32 ones).
constexpr int kControlRegs = 56, kEpilogueRegs = 224;
static_assert(128 * kControlRegs + 256 * kEpilogueRegs <= kLaunchThreads * 168, "register split");     // checked at the first launch too

// kind::f8f6f4 with e4m3 operands (format code 0) and f32 accumulation has the same fields as kind::f16.
constexpr uint32_t make_idesc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CTA_GROUP>
__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                           uint32_t idesc, uint32_t accumulate) {
    if (CTA_GROUP == 1)
        asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %6, 0;\n"
                     "mov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
                     "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n}"
                     :: "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %6, 0;\n"
                     "mov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
                     "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p;\n}"
                     :: "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}

// Arrival at a barrier of the pair's leader with release at CTA scope: what it publishes is the end of
// TMEM reads (ordered by tcgen05.fence), no memory writes, and the cluster-scope release of
// mbar_arrive_cluster costs the warp about 1400 clocks on each block.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(bar_cluster_addr) : "memory");
}

struct Shape {
    int m;                // rows of A and D (grouped: capacity)
    int n;
    int blocks;           // scale blocks of K
    int tiles_m;
    int tiles_n;
    int band;             // M-tiles per raster band
    int experts;          // 0 = dense
    int n_blocks;         // scale blocks of N (of one expert)
    int split;            // CTAs of a cluster that share a tile, each with a part of K
};

struct TilePos {
    int row0, row_end, col0, expert;
};

// BN = 256: a pair of CTAs works on 256 x 256 tiles (cta_group::2).  BN = 128: one CTA, 128 x 128 tiles, or
// (ROWS = 32) 32 x 128 ones for products with few rows: A's share of a stage shrinks from 16 to 4 KiB, so that
// ten stages fit instead of four and the weight streams with 160 KiB of it in flight.  The MMA still takes 128
// rows; the ones past the 32nd read the bytes behind them in the same stage and land in TMEM lanes that nobody
// reads.
template <int BN, int ROWS, typename OutT>
__global__ void __launch_bounds__(ROWS == 32 ? kFewThreads : kLaunchThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a_small,
                const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_d, const float* __restrict__ a_scale,
                const float* __restrict__ b_scale, const int* __restrict__ offsets, OutT* __restrict__ out, Shape shape,
                int* status, int kernel_id) {
    constexpr int CTA_GROUP = BN / 128;
    constexpr int kHalves = BN / kAccCols;                    // accumulators of a block: one for each 128 columns
    constexpr int kABytes = ROWS * BK;
    constexpr bool kFew = ROWS < BM;
    constexpr int kThreads = kFew ? kFewThreads : kLaunchThreads;
    constexpr int kEpiWarps = kFew ? 2 : 8;
    constexpr int kAccs = 4;                                  // accumulators: all of TMEM
    constexpr int kProducer = kFew ? 2 : 0;                   // warp roles; warp 1 issues MMAs, warp 3 copies scales
    constexpr int kBRows = kAccCols / CTA_GROUP;              // rows of B_T this CTA loads for an accumulator
    constexpr int kStage = kABytes + kHalves * kBRows * BK;
    constexpr int kOutBytes = kFew ? 0 : kEpiWarps * kBoxes * kBoxBytes;      // few rows are stored directly
    static_assert(kRingBytes - kOutBytes >= ROWS * kPartPitch * 4, "partial tile");
    constexpr int kStages = (kRingBytes - kOutBytes) / kStage, kStagesAll = kRingBytes / kStage;
    static_assert(kStage >= BM * BK, "the MMA reads 128 rows of A from its stage");
    constexpr int kTileRows = ROWS * CTA_GROUP;
    constexpr uint32_t kTmemCols = kAccs * kAccCols;
    constexpr uint32_t kIdesc = make_idesc_e4m3(BM * CTA_GROUP, kAccCols);
    constexpr int kCols = BN / 2;                             // columns of an epilogue warp: f32 sums of a thread
    constexpr int kColBlocks = BN / BK;                       // scale blocks of a tile's columns

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t s_ring = smem_base;
    const uint32_t s_bar = s_ring + kRingBytes + kTableBytes + kScaleBytes;
    int* seg = reinterpret_cast<int*>(smem_gen + kRingBytes);      // [experts+1] row offsets
    int* seg_tile = seg + kMaxExperts + 1;                    // [experts+1] M-tiles before
    const uint32_t s_scales = s_ring + kRingBytes + kTableBytes;      // 2 x ([kGroup][BM] of A, [kColBlocks][kGroup] of B)
    const float* scales = reinterpret_cast<const float*>(smem_gen + (s_scales - smem_base));
    const uint32_t bar_full = s_bar, bar_empty = bar_full + 8 * kStagesAll;
    const uint32_t bar_tfull = bar_empty + 8 * kStagesAll, bar_tempty = bar_tfull + 8 * kAccs;
    const uint32_t bar_sfull = bar_tempty + 8 * kAccs, bar_sempty = bar_sfull + 16;
    const uint32_t s_tmem_slot = bar_sempty + 16, s_abort = s_tmem_slot + 8;
    int4* tile_at = reinterpret_cast<int4*>(smem_gen + (s_bar - smem_base) + 512);      // [2], beside the scales
    volatile uint32_t* tmem_slot_gen = (volatile uint32_t*)(smem_gen + (s_tmem_slot - smem_base));
    volatile int* abort_gen = (volatile int*)(smem_gen + (s_abort - smem_base));

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t pair_rank = CTA_GROUP == 2 ? cluster_ctarank() : 0u;
    const int split = BN == 128 ? shape.split : 1;            // only the 128-column form splits K
    const int split_rank = split > 1 ? (int)cluster_ctarank() : 0;
    const int unit = (int)blockIdx.x / (split * CTA_GROUP), n_units = (int)gridDim.x / (split * CTA_GROUP);
    // this CTA's scale blocks of K
    const int kb0 = (int)((long long)shape.blocks * split_rank / split);
    const int kb1 = (int)((long long)shape.blocks * (split_rank + 1) / split);
    WaitCtx ctx{status, abort_gen, kernel_id};

    if (threadIdx.x == 0) {
        *abort_gen = 0;
        for (int s = 0; s < kStagesAll; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < kAccs; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, kEpiWarps / kHalves * CTA_GROUP);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_sfull + 8 * b, 33);                // 32 lanes' copies, and the tile's position
            mbar_init(bar_sempty + 8 * b, kEpiWarps);
        }
        fence_mbarrier_init();
        fence_proxy_async_smem();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        prefetch_tmap(&tmap_d);
    }
    if (warp == 1) {
        tmem_alloc<CTA_GROUP>(s_tmem_slot, kTmemCols);
        tmem_relinquish<CTA_GROUP>();
    }
    pdl_launch_dependents();
    const bool grouped = shape.experts > 0;
    if (grouped) pdl_wait();
    if (grouped && warp == 0) {
        // Row offsets, made non-decreasing and clipped to [0, m] whatever they hold, and the number of
        // M-tiles before each expert; 32 experts at a time.
        int run_max = 0, run_tiles = 0;
        const int first = min(max(__ldg(offsets), 0), shape.m);
        run_max = first;
        if (lane == 0) { seg[0] = first; seg_tile[0] = 0; }
        for (int e0 = 0; e0 < shape.experts; e0 += 32) {
            const int e = e0 + lane;
            int end = e < shape.experts ? min(max(__ldg(offsets + e + 1), 0), shape.m) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, end, o);
                if (lane >= o) end = max(end, v);
            }
            end = max(end, run_max);
            int start = __shfl_up_sync(0xffffffffu, end, 1);
            if (lane == 0) start = run_max;
            int tiles = (end - start + kTileRows - 1) / kTileRows;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, tiles, o);
                if (lane >= o) tiles += v;
            }
            tiles += run_tiles;
            if (e < shape.experts) { seg[e + 1] = end; seg_tile[e + 1] = tiles; }
            run_max = __shfl_sync(0xffffffffu, end, 31);
            run_tiles = __shfl_sync(0xffffffffu, tiles, 31);
        }
    }
    tc_fence_before_sync();
    if (CTA_GROUP == 2) cluster_sync_all(); else __syncthreads();
    tc_fence_after_sync();
    // Set-up above overlaps the previous kernel's tail; global memory is read and written only below.
    if (!grouped) pdl_wait();
    const uint32_t tmem_base = *tmem_slot_gen;
    const int n_tiles = (grouped ? seg_tile[shape.experts] : shape.tiles_m) * shape.tiles_n;
    // A 128-column tile whose CTA has no other has no loads left when it is stored, and its last accumulator says that
    // its MMAs have read the ring, so the store boxes' memory serves the ring until then.  With four stages a block
    // takes a quarter of a stage's way (864 ns from load to MMA, 384 back); with six 512 x 4096 x 4096 from HBM takes
    // 11.7 us instead of 12.9.  (A pair would have to wait for its other half's MMAs: 768 x 4096 x 4096 17.5 us
    // instead of 17.05.)
    const int stages = BN == 128 && n_tiles <= n_units ? kStagesAll : kStages;

    auto tile_pos = [&](int t) {
        TilePos p;
        if (grouped) {
            int lo = 0, hi = shape.experts;          // last expert whose first tile is at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (seg_tile[mid] * shape.tiles_n <= t) lo = mid; else hi = mid;
            }
            const int r = t - seg_tile[lo] * shape.tiles_n, width = seg_tile[lo + 1] - seg_tile[lo];
            const int tn = r / width;                // an expert's M-tiles share a block of weights: M fastest
            p.expert = lo;
            p.row0 = seg[lo] + (r - tn * width) * kTileRows;
            p.row_end = seg[lo + 1];
            p.col0 = tn * BN;
        } else {
            const int band_tiles = shape.band * shape.tiles_n;
            const int b = t / band_tiles, r = t - b * band_tiles;
            const int m0 = b * shape.band, width = min(shape.band, shape.tiles_m - m0);
            const int tn = r / width;
            p.expert = 0;
            p.row0 = (m0 + r - tn * width) * kTileRows;
            p.row_end = shape.m;
            p.col0 = tn * BN;
        }
        return p;
    };

    if (kFew ? warp > 0 && warp < 4 : warp < 4) {
        if (BN == 256) reg_dealloc<kControlRegs>();
        if (warp == kProducer && lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            const uint32_t full_leader = CTA_GROUP == 2 ? map_to_cta(bar_full, 0) : bar_full;
            bool ok = true;
            for (int t = unit; t < n_tiles && ok; t += n_units) {
                const TilePos p = tile_pos(t);
                const int row_a = p.row0 + (int)pair_rank * BM;
                const bool small = kFew || p.row_end - row_a <= kSmallRows;
                const int row_b = p.expert * shape.n + p.col0 + (int)pair_rank * kBRows;      // of the first half
                // bytes of this CTA's loads, and for the leader of a pair its peer's too
                uint32_t tx = 0;
#pragma unroll
                for (int c = 0; c < CTA_GROUP; ++c)
                    tx += (uint32_t)((kFew || p.row_end - p.row0 - c * BM <= kSmallRows ? kSmallRows * BK : kABytes) + kHalves * kBRows * BK);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, ctx, 1))) break;
                    const uint32_t dst = s_ring + stage * kStage, bar = bar_full + 8 * stage;
                    if (CTA_GROUP == 1) {
                        mbar_arrive_expect_tx(bar, tx);
                        tma_load_2d(dst + kABytes, &tmap_b, bar, kb * BK, row_b);
                        tma_load_2d(dst, !kFew && small ? &tmap_a_small : &tmap_a, bar, kb * BK, row_a);
                    } else {
                        if (pair_rank == 0) mbar_arrive_expect_tx(bar, tx);
#pragma unroll
                        for (int h = 0; h < kHalves; ++h)
                            tma_load_2d_pair(dst + kABytes + h * kBRows * BK, &tmap_b, full_leader + 8 * stage, kb * BK, row_b + h * kAccCols);
                        tma_load_2d_pair(dst, small ? &tmap_a_small : &tmap_a, full_leader + 8 * stage, kb * BK, row_a);
                    }
                    if (++stage == stages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        if (warp == 1 && pair_rank == 0 && unit < n_tiles) {
            // The whole warp runs the loop and one elected lane issues (see elect_one): with descriptors in
            // uniform registers an MMA issues in a few clocks, from a lane's own registers in about 60, which is
            // as long as it executes, so that every wait would be a hole in the tensor pipe.
            const int total = ((n_tiles - unit - 1) / n_units + 1) * (kb1 - kb0);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            const uint64_t da0 = make_desc_kmajor_sw128(s_ring), db0 = make_desc_kmajor_sw128(s_ring + kABytes);
            const uint32_t a_hi = (uint32_t)(da0 >> 32), b_hi = (uint32_t)(db0 >> 32);
            const bool leader = elect_one();
            // The tensor pipe holds only a few MMAs, so that anything between one half's last and the next one's first
            // drains it: the next barriers are looked at, and the lanes' answers joined, before this half's last MMA
            // (a vote and two branches less between halves: 8192 x 8192 x 4096 194 -> 187 us on zeros).
            bool ok = true, ready = false;
            for (int i = 0; i < total && ok; ++i) {
                const uint32_t a_lo = (uint32_t)da0 + (uint32_t)(stage * (kStage >> 4));
                const uint32_t b_lo = (uint32_t)db0 + (uint32_t)(stage * (kStage >> 4));
                const uint32_t empty = bar_empty + 8 * stage, full = bar_full + 8 * stage, full_phase = phase;
                if (++stage == stages) { stage = 0; phase ^= 1u; }
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const uint32_t d = tmem_base + (uint32_t)(acc * kAccCols), tfull = bar_tfull + 8 * acc;
                    if (!ready) {
                        if (h == 0) ok = mbar_wait(full, full_phase, ctx, 3);
                        if (ok) ok = mbar_wait(bar_tempty + 8 * acc, acc_phase ^ 1u, ctx, 2);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                    }
                    tc_fence_after_sync();
                    const uint32_t b_half = b_lo + (uint32_t)(h * (kBRows * BK >> 4));
                    if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
                    // 32 e4m3 along K = 32 bytes = +2 in the encoded address
                    if (leader) {
                        umma_f8_ss<CTA_GROUP>(d, a_lo, a_hi, b_half, b_hi, kIdesc, 0u);
                        umma_f8_ss<CTA_GROUP>(d, a_lo + 2, a_hi, b_half + 2, b_hi, kIdesc, 1u);
                        umma_f8_ss<CTA_GROUP>(d, a_lo + 4, a_hi, b_half + 4, b_hi, kIdesc, 1u);
                    }
                    ready = mbar_test_wait(bar_tempty + 8 * acc, acc_phase ^ 1u);
                    if (h == kHalves - 1) ready = mbar_test_wait(bar_full + 8 * stage, phase) && ready;
                    ready = __all_sync(0xffffffffu, ready);
                    if (leader) {
                        umma_f8_ss<CTA_GROUP>(d, a_lo + 6, a_hi, b_half + 6, b_hi, kIdesc, 1u);
                        if (CTA_GROUP == 2) umma_commit_pair(tfull); else umma_commit<1>(tfull);
                        if (h == kHalves - 1) {
                            if (CTA_GROUP == 2) umma_commit_pair(empty); else umma_commit<1>(empty);
                        }
                    }
                }
            }
            __syncwarp();
        }
        if (warp == 3) {
            // Scales: this warp copies a group of blocks ahead into shared memory (four rows a lane), so that
            // no epilogue warp waits for global memory.
            int buf = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = unit; t < n_tiles && ok; t += n_units) {
                const TilePos p = tile_pos(t);
                const int row0 = p.row0 + (int)pair_rank * BM + lane;
                // lane c * kGroup + i copies block i's scale of column block c
                const int cb = lane / kGroup, ib = lane % kGroup;
                const bool b_there = cb < kColBlocks && p.col0 + cb * BK < shape.n;
                const float* sb = b_scale + ((long long)p.expert * shape.n_blocks + p.col0 / BK + (b_there ? cb : 0)) * shape.blocks;
                for (int kb = kb0; kb < kb1; kb += kGroup) {
                    ok = mbar_wait(bar_sempty + 8 * buf, phase ^ 1u, ctx, 5);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t dst = s_scales + (uint32_t)(buf * kScaleWords + lane) * 4u;
#pragma unroll 1
                    for (int j = 0; j < ROWS / 32; ++j) {
                        const bool there = row0 + 32 * j < p.row_end;
                        const float* sa = a_scale + (there ? (long long)(row0 + 32 * j) * shape.blocks : 0ll);
#pragma unroll
                        for (int i = 0; i < kGroup; ++i)      // blocks past the end: any word of the row, never used
                            cp_async_4(dst + (uint32_t)(i * BM + 32 * j) * 4u, sa + min(kb + i, kb1 - 1), there);
                    }
                    if (lane < 2 * kGroup) cp_async_4(dst + kGroup * BM * 4u, sb + min(kb + ib, kb1 - 1), b_there);
                    cp_async_arrive(bar_sfull + 8 * buf);
                    if (lane == 0) {
                        // the epilogue takes the tile's position from here instead of working it out between tiles
                        tile_at[buf] = make_int4(p.row0, p.row_end, p.col0, p.expert);
                        mbar_arrive(bar_sfull + 8 * buf);
                    }
                    if (++buf == 2) { buf = 0; phase ^= 1u; }
                }
            }
            cp_async_wait_all();
        }
    } else if (!kFew || warp == 0 || warp == 4) {
        if (BN == 256) reg_alloc<kEpilogueRegs>();
        const int q = warp & 3, group = kFew ? warp >> 2 : (warp - 4) >> 2;      // few rows: warps 0 and 4
        const uint32_t box = s_ring + kRingBytes - kOutBytes + (kFew ? 0u : (uint32_t)(warp - 4) * (kBoxes * kBoxBytes));
        const uint32_t tempty_leader = CTA_GROUP == 2 ? map_to_cta(bar_tempty, 0) : bar_tempty;
        constexpr int kAccStep = kHalves;            // this warp's accumulators: those of its half
        static_assert(kAccs % kHalves == 0, "a half's accumulators");
        const int acc0 = kHalves == 2 ? group : 0, col_in_acc = kHalves == 2 ? 0 : group * kCols;
        int acc = acc0, sbuf = 0;
        uint32_t acc_phase = 0, sphase = 0;
        bool ok = true, seen = false;                // seen: the next accumulator was complete at the last look
        for (int t = unit; t < n_tiles && ok; t += n_units) {
            float sum[kCols];
#pragma unroll
            for (int i = 0; i < kCols; ++i) sum[i] = 0.0f;
            for (int kb = kb0; kb < kb1 && ok; kb += kGroup) {
                ok = mbar_wait(bar_sfull + 8 * sbuf, sphase, ctx, 6);
                const float* sa = scales + sbuf * kScaleWords + q * 32 + lane;
                const float* sb = scales + sbuf * kScaleWords + kGroup * BM + group * kCols / BK * kGroup;
                const int n_blocks = min(kGroup, kb1 - kb);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                float s_next = sa[0] * sb[0];
                for (int i = 0; i < n_blocks; ++i) {
                    // A block is a chain of latencies for this warp, so whatever can leaves the chain: the scale is
                    // read a block ahead, and the next accumulator's barrier looked at under the last FMAs.
                    const float s = s_next;
                    if (!__all_sync(0xffffffffu, seen)) {
                        ok = mbar_wait(bar_tfull + 8 * acc, acc_phase, ctx, 4);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                    }
                    tc_fence_after_sync();
                    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kAccCols + col_in_acc);
                    // The accumulator is handed back once its last columns are in registers: two batches of loads
                    // (tcgen05.wait::ld waits for all that are in flight), the second under the FMAs of the first.
                    constexpr int kChunks = kCols / 32;
                    static_assert(kChunks == 2 || kChunks == 4, "two batches");
                    uint32_t v[2][32];
                    tmem_ld_32x32b_x32(t_row, v[0]);
                    tmem_ld_32x32b_x32(t_row + 32, v[1]);
                    tmem_ld_wait();
                    reg_fence(v[0]);
                    reg_fence(v[1]);
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        if (c == kChunks - 2) {
                            if (kChunks > 2) { tmem_ld_wait(); reg_fence(v[0]); reg_fence(v[1]); }
                            tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0) {
                                if (CTA_GROUP == 2) mbar_arrive_remote(tempty_leader + 8 * acc);
                                else mbar_arrive(bar_tempty + 8 * acc);
                            }
                            if ((acc += kAccStep) >= kAccs) { acc = acc0; acc_phase ^= 1u; }
                            const int next = min(i + 1, n_blocks - 1);
                            s_next = sa[next * BM] * sb[next];
                        }
                        if (c == kChunks - 1) seen = mbar_test_wait(bar_tfull + 8 * acc, acc_phase);
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            fma2v(sum[c * 32 + j], sum[c * 32 + j + 1], __uint_as_float(v[c & 1][j]), __uint_as_float(v[c & 1][j + 1]),
                                  s, s, sum[c * 32 + j], sum[c * 32 + j + 1]);
                        if (c + 2 < kChunks) {
                            reg_fence(v[c & 1]);
                            tmem_ld_32x32b_x32(t_row + (c + 2) * 32, v[c & 1]);
                        }
                    }
                }
                if (kb + kGroup >= kb1) break;               // the tile's last group is handed back below
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_sempty + 8 * sbuf);
                if (++sbuf == 2) { sbuf = 0; sphase ^= 1u; }
            }
            if (!ok) break;
            const int4 at = tile_at[sbuf];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_sempty + 8 * sbuf);
            if (++sbuf == 2) { sbuf = 0; sphase ^= 1u; }
            const TilePos p{at.x, at.y, at.z, at.w};
            const int row_limit = kFew ? min(p.row_end, p.row0 + ROWS) : p.row_end;
            const int row = p.row0 + (int)pair_rank * BM + q * 32 + lane;      // this thread's row
            const int col = p.col0 + group * kCols;                   // this warp's first column
            if (split > 1) {
                // One tile a cluster: the ring is drained (every MMA that read it has been waited for
                // through its accumulator), so the partial tile goes there.
                float* mine = reinterpret_cast<float*>(smem_gen) + (q * 32 + lane) * kPartPitch + group * kCols;
                if (row < row_limit) {
#pragma unroll
                    for (int i = 0; i < kCols; i += 4)
                        *reinterpret_cast<float4*>(mine + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
                }
                break;
            }
            constexpr int kBoxCols = 128 / (int)sizeof(OutT);
            const int row_w = p.row0 + (int)pair_rank * BM + q * 32;      // first row of this warp
            // TMA clips a box at the matrix's edges, but not at the end of an expert's rows.
            // A tile's boxes go round the buffers; with fewer boxes than buffers every tile starts at the same one.
            constexpr int kBoxesBehind = kCols / kBoxCols >= kBoxes ? kBoxes - 1 : 0;
            static_assert(kBoxesBehind == 0 || kCols / kBoxCols % kBoxes == 0, "a tile ends where it began");
            const bool whole = !kFew && (shape.experts == 0 || row_w + 32 <= p.row_end);
#pragma unroll
            for (int c = 0; c < kCols / kBoxCols; ++c) {
                uint32_t w[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (sizeof(OutT) == 4) {
                        w[i] = __float_as_uint(sum[c * kBoxCols + i]);
                    } else {
                        __nv_bfloat162 b2 = __floats2bfloat162_rn(sum[(c * kBoxCols + 2 * i) % kCols], sum[(c * kBoxCols + 2 * i + 1) % kCols]);
                        w[i] = *reinterpret_cast<uint32_t*>(&b2);
                    }
                }
                if (whole) {
                    const uint32_t buf = box + (uint32_t)(c % kBoxes) * kBoxBytes;
                    if (lane == 0) tma_store_wait_read<kBoxesBehind>();      // the store that last read this buffer
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        st_shared_v4(buf + (uint32_t)(lane * 128 + ((j ^ (lane & 7)) << 4)), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (row_w < p.row_end && col + c * kBoxCols < shape.n) tma_store_2d(&tmap_d, buf, col + c * kBoxCols, row_w);
                        tma_store_commit();
                    }
                } else if (row < row_limit) {
                    OutT* dst = out + (long long)row * shape.n + col + c * kBoxCols;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + c * kBoxCols + j * (16 / (int)sizeof(OutT)) < shape.n)
                            reinterpret_cast<uint4*>(dst)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
            }
        }
        if (lane == 0) tma_store_wait_read<0>();      // shared memory must outlive the stores' reads
    }

    __syncwarp();
    tc_fence_before_sync();
    if (split > 1) {
        // Sum of the partial tiles, read through distributed shared memory in the order of K: CTA r of the
        // cluster finishes every split-th vector of the tile.  (Writing the partial sums to the CTA that adds
        // them needs one barrier less here but one more at the start, and measured 0.6 us slower.)
        cluster_sync_all();
        if (unit < n_tiles) {
            const TilePos p = tile_pos(unit);
            const int rows = min(ROWS, p.row_end - p.row0), vecs = BN / 4;
            uint32_t peer[kMaxSplit];
#pragma unroll
            for (int s = 0; s < kMaxSplit; ++s) peer[s] = map_to_cta(smem_base, (uint32_t)min(s, split - 1));
            for (int i = split_rank * kThreads + (int)threadIdx.x; i < rows * vecs; i += split * kThreads) {
                const int r = i / vecs, c = (i - r * vecs) * 4;
                float4 v[kMaxSplit];
#pragma unroll
                for (int s = 0; s < kMaxSplit; ++s)
                    if (s < split)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
                                     : "r"(peer[s] + (uint32_t)(r * kPartPitch + c) * 4u) : "memory");
                float4 sum = v[0];
#pragma unroll
                for (int s = 1; s < kMaxSplit; ++s)
                    if (s < split) { sum.x += v[s].x; sum.y += v[s].y; sum.z += v[s].z; sum.w += v[s].w; }
                if (p.col0 + c < shape.n) {
                    OutT* dst = out + (long long)(p.row0 + r) * shape.n + p.col0 + c;
                    if (sizeof(OutT) == 4) {
                        *reinterpret_cast<float4*>(dst) = sum;
                    } else {
                        __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
                        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
                    }
                }
            }
        }
        cluster_sync_all();
    } else if (CTA_GROUP == 2) {
        cluster_sync_all();
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc<CTA_GROUP>(tmem_base, kTmemCols);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile shape and split of K.
//   8 rows at most, dense: the streaming kernel of fp8_gemm_skinny.cu (1 x 4096 x 4096 from HBM: 4.9 us against
//   7.0 on 32 x 128 tiles), with 9 to 16 rows up to 16 Mi weights, since its arithmetic doubles (16 x 4096 x 4096:
//   6.4 against 7.4 us, but 16 x 8192 x 8192: 19.5 against 15), and with 17 to 32 rows up to 4 Mi weights where a warp
//   has one block of K (32 x 2048 x 2048: 4.5 against 5.8 us, 32 x 1024 x 1024: 3.6 against 4.4; but 32 x 4096 x 2048
//   6.2 against 6.1 and 32 x 1024 x 4096, two blocks a warp, 6.7 against 5.7).
//   few rows: 32 x 128 tiles; dense up to 32 rows (32 x 4096 x 4096: 7.5 us, on 128 x 128 tiles 7.7), grouped up to 24
//   for each expert on average, since loads are uneven (32 experts, 4096 x 2048: 24 rows 48.6 us, on 128 x 128 tiles
//   52.3; 28 rows 54.5 and 52.8).
//   dense: 128 x 128 tiles while they fit the SMs at once (512 x 4096 x 4096: 11.6 us, as pairs 16.2), else
//   256 x 256 tiles of CTA pairs (768 x 4096 x 4096: 17.0 us, as 128 x 128 ones one after the other 21.3),
//   unless a pair's tile would be half empty (40000 x 128 x 4096: 42 us, as pairs 50).  Where 128-column tiles
//   leave SMs idle the K blocks of a tile, if they are 20 or more, are shared by a cluster of up to 8 CTAs (at
//   least eight blocks each: the cluster's two barriers take about 1.6 us), which add their partial tiles through
//   distributed shared memory in a fixed order (256 rows and 2048 x 2048: 6.9 us, shared by two 7.5; 64 rows and
//   2048 x 3584: 9.1 and 7.8; 64 rows and 4096 x 4096: by two 8.9, by four 8.4).
//   grouped: the tiles are known on the device only, so the rows an expert can have on average decide (the capacity:
//   the figures have buffers that are full; 64 experts of 2 rows in 8192 rows take 63 us, in 128 rows 45): pairs from
//   128 (32 experts, 4096 x 2048: 96 rows 60 us on 128 x 128 tiles, 71 as pairs; 128 rows 74.7 and 72.2; 200 rows
//   92 and 75).
struct Plan {
    int64_t experts, m, n, k, tiles;
    int bn, rows, split;
    bool skinny;
    int cta_group() const { return bn / 128; }
};

Plan make_plan(const Record& r) {
    Plan p{};
    const bool grouped = r.kernel_id == PB200_K_FP8_GROUPED_GEMM;
    const int64_t* d = r.dims + (grouped ? 1 : 0);
    p.experts = grouped ? r.dims[0] : 0;
    p.m = d[0]; p.n = d[1]; p.k = d[2];
    p.split = 1;
    const int64_t sms = sm_count(), mean_rows = grouped ? ceil_div(p.m, p.experts) : p.m;
    if (!grouped && (p.m <= 8 || (p.m <= 16 && p.n * p.k <= (1 << 24)) ||
                     (p.m <= 32 && p.n * p.k <= (1 << 22) && ceil_div(p.k, BK) <= fp8_skinny_warps(p.n, p.k)))) {
        p.skinny = true;
        p.tiles = fp8_skinny_grid(p.n);
        return p;
    }
    if (mean_rows <= (grouped ? kSmallRows * 3 / 4 : kSmallRows)) { p.bn = 128; p.rows = kSmallRows; }
    else if (p.n > 128 && (grouped ? mean_rows >= BM : ceil_div(p.m, BM) * ceil_div(p.n, 128) > sms)) { p.bn = 256; p.rows = BM; }
    else { p.bn = 128; p.rows = BM; }
    // every expert may end in a partial tile
    p.tiles = (ceil_div(p.m, p.rows * p.cta_group()) + p.experts) * ceil_div(p.n, p.bn);
    if (!grouped && p.bn == 128) {
        const int64_t blocks = ceil_div(p.k, BK);
        // A cluster lives in one GPC, so only so many run at once: 15 of 8 CTAs and 33 of 4 were seen to (a
        // 16th doubles 32 x 2048 x 8192 from 8.0 to 13.6 us), and GPUs differ in which SMs they have.
        auto fits = [&](int64_t split) { return p.tiles * split <= (split == 8 ? sms * 3 / 4 : split == 4 ? sms * 7 / 8 : sms); };
        while (p.split < kMaxSplit && fits(p.split * 2) && blocks >= (p.split == 1 ? 20 : 16 * p.split)) p.split *= 2;
    }
    return p;
}

// CTAs of a launch: whole clusters, one for each tile or as many as the SMs hold.
int64_t grid_of(const Plan& p) {
    const int64_t cluster = p.split * p.cta_group(), most = p.split > 1 ? p.tiles : sm_count() / p.cta_group();
    return (p.tiles < most ? p.tiles : most) * cluster;
}

int threads_of(int rows) { return rows == kSmallRows ? kFewThreads : kLaunchThreads; }

template <int BN, int ROWS, typename OutT>
int launch_variant(const Record& r, const Plan& p, cudaStream_t stream, void** ptrs, char* err) {
    constexpr int CTA_GROUP = BN / 128;
    auto kernel = fp8_gemm_kernel<BN, ROWS, OutT>;
    static std::atomic<uint64_t> attr_set{0};   // bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(attr_set.load(std::memory_order_relaxed) & (1ull << (dev & 63)))) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemTotal);
        if (e != cudaSuccess) { set_err(err, "cudaFuncSetAttribute(smem=%d): %s", kSmemTotal, cudaGetErrorString(e)); return PB200_ERR_LAUNCH; }
        // The register split of the 256-column form draws on what the launch gets; with fewer it would wait for ever.
        cudaFuncAttributes fa{};
        e = cudaFuncGetAttributes(&fa, kernel);
        if (e != cudaSuccess || (BN == 256 && fa.numRegs * kLaunchThreads < 128 * kControlRegs + 256 * kEpilogueRegs)) {
            set_err(err, "fp8 gemm: %d registers a thread are too few for its register split", fa.numRegs);
            return PB200_ERR_LAUNCH;
        }
        attr_set.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
    auto map = [&](CUtensorMap* m, const void* base, int64_t rows, uint32_t box_rows) {
        uint64_t dims[2] = {(uint64_t)p.k, (uint64_t)rows};
        uint64_t str[1] = {(uint64_t)p.k};
        uint32_t box[2] = {BK, box_rows};
        return make_tensor_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, err);
    };
    CUtensorMap ta, ta_small, tb;
    if (int rc = map(&ta, ptrs[0], p.m, ROWS)) return rc;
    if (int rc = map(&ta_small, ptrs[0], p.m, kSmallRows)) return rc;
    if (int rc = map(&tb, ptrs[2], p.n * (p.experts ? p.experts : 1), kAccCols / CTA_GROUP)) return rc;
    CUtensorMap td;
    {
        uint64_t dims[2] = {(uint64_t)p.n, (uint64_t)p.m};
        uint64_t str[1] = {(uint64_t)p.n * sizeof(OutT)};
        uint32_t box[2] = {128 / sizeof(OutT), 32};
        if (int rc = make_tensor_map(&td, sizeof(OutT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                     ptrs[p.experts ? 5 : 4], dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, err)) return rc;
    }
    Shape s;
    s.m = (int)p.m;
    s.n = (int)p.n;
    s.blocks = (int)ceil_div(p.k, BK);
    s.tiles_m = (int)ceil_div(p.m, ROWS * CTA_GROUP);
    s.tiles_n = (int)ceil_div(p.n, BN);
    s.band = s.tiles_m < 16 ? s.tiles_m : 16;
    s.experts = (int)p.experts;
    s.n_blocks = (int)ceil_div(p.n, BK);
    s.split = p.split;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid_of(p));
    cfg.blockDim = dim3(threads_of(ROWS));
    cfg.dynamicSmemBytes = kSmemTotal;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)(p.split * CTA_GROUP);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.split * CTA_GROUP > 1 ? 2 : 1;
    const bool grouped = p.experts > 0;
    const int* offsets = grouped ? (const int*)ptrs[4] : nullptr;
    OutT* out = (OutT*)ptrs[grouped ? 5 : 4];
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ta, ta_small, tb, td, (const float*)ptrs[1], (const float*)ptrs[3], offsets, out, s,
                                       device_status_ptr(), (int)r.kernel_id);
    if (e != cudaSuccess) {
        set_err(err, "fp8 gemm launch failed (BN=%d cta_group=%d split=%d): %s", BN, CTA_GROUP, p.split, cudaGetErrorString(e));
        return p.split * CTA_GROUP > 1 ? PB200_ERR_CLUSTER : PB200_ERR_LAUNCH;
    }
    return PB200_OK;
}

}  // namespace

int plan_fp8_gemm(Record& r, char* err) {
    const bool grouped = r.kernel_id == PB200_K_FP8_GROUPED_GEMM;
    const int need = grouped ? 4 : 3;
    if (r.n_dims != need) { set_err(err, "kernel %d needs %d dims, got %d", r.kernel_id, need, r.n_dims); return PB200_ERR_BAD_SHAPE; }
    for (int i = 0; i < need; ++i) {
        if (r.dims[i] < 1) { set_err(err, "G, M, N, K must be positive"); return PB200_ERR_BAD_SHAPE; }
        if (r.dims[i] > 0x7fffffffLL) { set_err(err, "extent exceeds 2^31-1"); return PB200_ERR_BAD_SHAPE; }
    }
    if (grouped && r.dims[0] > kMaxExperts) { set_err(err, "G=%lld exceeds %d", (long long)r.dims[0], kMaxExperts); return PB200_ERR_BAD_SHAPE; }
    const Plan p = make_plan(r);
    if (p.n % 8 != 0) { set_err(err, "N=%lld must be divisible by 8", (long long)p.n); return PB200_ERR_BAD_SHAPE; }
    if (p.k % 16 != 0) { set_err(err, "K=%lld must be divisible by 16", (long long)p.k); return PB200_ERR_BAD_SHAPE; }
    // row coordinates of a tile run up to a tile past the last row
    if (p.m + 2 * BM > 0x7fffffffLL || (grouped ? p.experts : 1) * p.n + 256 > 0x7fffffffLL || p.k + BK > 0x7fffffffLL ||
        p.tiles > 0x3fffffffLL) {
        set_err(err, "extent exceeds 2^31-1");
        return PB200_ERR_BAD_SHAPE;
    }
    pb200_geometry& g = r.geom;
    g.n_inputs = grouped ? 5 : 4;
    g.n_outputs = 1;
    g.grid[1] = g.grid[2] = g.block[1] = g.block[2] = g.cluster[0] = g.cluster[1] = g.cluster[2] = 1;
    if (p.skinny) {
        g.grid[0] = (uint32_t)p.tiles;
        g.block[0] = (uint32_t)(32 * fp8_skinny_warps(p.n, p.k));
        g.smem_bytes = (uint32_t)fp8_skinny_smem(p.m, p.n, p.k);
        return PB200_OK;
    }
    g.grid[0] = (uint32_t)grid_of(p);
    g.block[0] = (uint32_t)threads_of(p.rows);
    g.cluster[0] = (uint32_t)(p.split * p.cta_group());
    g.smem_bytes = kSmemTotal;
    return PB200_OK;
}

int launch_fp8_gemm(const Record& r, cudaStream_t stream, void** ptrs, char* err) {
    const Plan p = make_plan(r);
    if (p.skinny) return launch_fp8_skinny(r, p.m, p.n, p.k, stream, ptrs, err);
    const bool b16 = (r.flags & PB200_F_OUT_BF16) != 0;
#define PB200_FP8_CASE(BN_, ROWS_)                                                                  \
    if (p.bn == BN_ && p.rows == ROWS_)                                                             \
        return b16 ? launch_variant<BN_, ROWS_, __nv_bfloat16>(r, p, stream, ptrs, err)             \
                   : launch_variant<BN_, ROWS_, float>(r, p, stream, ptrs, err);
    PB200_FP8_CASE(256, 128)
    PB200_FP8_CASE(128, 128)
    PB200_FP8_CASE(128, 32)
#undef PB200_FP8_CASE
    set_err(err, "no fp8 gemm variant for %d x %d tiles", p.rows, p.bn);
    return PB200_ERR_BAD_SHAPE;
}

}  // namespace pb200
