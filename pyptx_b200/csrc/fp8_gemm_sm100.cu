// Block-scaled e4m3 GEMM for sm_100a on the 5th-generation tensor cores:
//   D[m,n] = sum over 128-wide blocks b of K of
//            a_scale[m,b] * b_scale[n/128,b] * sum_{k in b} A[m,k] * B_T[n,k]
// dense (M, N, K) and grouped by device-side row offsets (expert e owns rows
// [offsets[e], offsets[e+1]) of A and D and its own N rows of B_T; any alignment).
//
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4, f32 accumulation in TMEM), one
// accumulator for each block of K; the scales are f32 and differ from row to row, so the outer sum
// runs in registers: eight epilogue warps fetch each block's accumulator from TMEM, multiply it by
// the row's scale times the weight block's and add it to the tile's f32 sums.  128 rows are the 128
// TMEM lanes, so a thread has one row: one scale for a block of K, and its columns lie in one weight
// block.
//
// What bounds it: a 128 x 256 x 128 block takes 512 clocks of MMA, and the drain of its accumulator
// 256 clocks of TMEM reads and 128 of packed FMA issue on each SM sub-partition.  Two accumulators
// in TMEM let the drain of one block run under the MMAs of the next.
//
// Structure as the bf16 GEMM's (gemm_sm100.cu): persistent, warp 0 = TMA producer, warp 1 = MMA
// issuer and TMEM owner, warps 4-11 = epilogue (two for each quarter of the lanes, each with half of
// the columns).  Bounded waits throughout.
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
constexpr int kThreads = 384;                // 12 warps: 4 of control, 8 of epilogue
constexpr int kEpiWarps = 8;
constexpr int kSmallRows = 32;               // row box of A for tiles with few rows
constexpr int kRing = 192 * 1024;            // operand ring
constexpr int kChunkBytes = 64;              // bytes of a row that a warp stages at a time
constexpr int kStageBytes = 32 * kChunkBytes;
constexpr int kMaxExperts = 1024;
constexpr int kTableBytes = 2 * (kMaxExperts + 1) * 4 + 120;      // sanitised offsets and tile prefix, padded to 128
constexpr int kBarBytes = 1024;
constexpr int kSmemTotal = 1024 + kRing + kEpiWarps * kStageBytes + kTableBytes + kBarBytes;
static_assert(kSmemTotal <= 227 * 1024, "shared memory");
constexpr int kMaxSplit = 8;
// Registers of the 256-column form, whose epilogue threads hold 128 sums: the launch has 384 x 168;
// the control warpgroup gives up 128 x 128 of them and the two epilogue warpgroups take 256 x 64.
constexpr int kControlRegs = 40, kEpilogueRegs = 232;
static_assert(128 * kControlRegs + 256 * kEpilogueRegs <= kThreads * 168, "register split");
constexpr int kPartPitch = 128 + 4;          // f32 row pitch of a split's partial tile: rows on distinct banks

// kind::f8f6f4 with e4m3 operands (format code 0) and f32 accumulation has the same fields as kind::f16.
constexpr uint32_t make_idesc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                           uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %6, 0;\n"
                 "mov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n}"
                 :: "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
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

template <int BN, typename OutT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a_small,
                const __grid_constant__ CUtensorMap tmap_b, const float* __restrict__ a_scale,
                const float* __restrict__ b_scale, const int* __restrict__ offsets, OutT* __restrict__ out, Shape shape,
                int* status, int kernel_id) {
    constexpr int kABytes = BM * BK;
    constexpr int kStage = kABytes + BN * BK;
    constexpr int kStages = kRing / kStage;
    constexpr int kAccs = 512 / BN > 4 ? 4 : 512 / BN;        // accumulators in TMEM
    constexpr uint32_t kTmemCols = kAccs * BN;
    constexpr uint32_t kIdesc = make_idesc_e4m3(BM, BN);
    constexpr int kCols = BN / 2;                             // columns of an epilogue warp

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t s_ring = smem_base;
    const uint32_t s_epi = s_ring + kRing;
    const uint32_t s_bar = s_epi + kEpiWarps * kStageBytes + kTableBytes;
    int* seg = reinterpret_cast<int*>(smem_gen + kRing + kEpiWarps * kStageBytes);     // [experts+1] row offsets
    int* seg_tile = seg + kMaxExperts + 1;                                             // [experts+1] M-tiles before
    const uint32_t bar_full = s_bar, bar_empty = bar_full + 8 * kStages;
    const uint32_t bar_tfull = bar_empty + 8 * kStages, bar_tempty = bar_tfull + 8 * kAccs;
    const uint32_t s_tmem_slot = bar_tempty + 8 * kAccs, s_abort = s_tmem_slot + 8;
    volatile uint32_t* tmem_slot_gen = (volatile uint32_t*)(smem_gen + (s_tmem_slot - smem_base));
    volatile int* abort_gen = (volatile int*)(smem_gen + (s_abort - smem_base));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = BN == 128 ? shape.split : 1;            // only the 128-column form splits K
    const int split_rank = split > 1 ? (int)cluster_ctarank() : 0;
    const int unit = (int)blockIdx.x / split, n_units = (int)gridDim.x / split;
    // this CTA's scale blocks of K
    const int kb0 = (int)((long long)shape.blocks * split_rank / split);
    const int kb1 = (int)((long long)shape.blocks * (split_rank + 1) / split);
    WaitCtx ctx{status, abort_gen, kernel_id};

    if (threadIdx.x == 0) {
        *abort_gen = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < kAccs; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, kEpiWarps);
        }
        fence_mbarrier_init();
        fence_proxy_async_smem();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    if (warp == 1) {
        tmem_alloc<1>(s_tmem_slot, kTmemCols);
        tmem_relinquish<1>();
    }
    pdl_launch_dependents();
    pdl_wait();
    if (shape.experts > 0 && warp == 0) {
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
            int tiles = (end - start + BM - 1) / BM;
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
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_gen;
    const int n_tiles = (shape.experts > 0 ? seg_tile[shape.experts] : shape.tiles_m) * shape.tiles_n;

    auto tile_pos = [&](int t) {
        TilePos p;
        if (shape.experts > 0) {
            int lo = 0, hi = shape.experts;          // last expert whose first tile is at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (seg_tile[mid] * shape.tiles_n <= t) lo = mid; else hi = mid;
            }
            const int r = t - seg_tile[lo] * shape.tiles_n, width = seg_tile[lo + 1] - seg_tile[lo];
            const int tn = r / width;                // an expert's M-tiles share a block of weights: M fastest
            p.expert = lo;
            p.row0 = seg[lo] + (r - tn * width) * BM;
            p.row_end = seg[lo + 1];
            p.col0 = tn * BN;
        } else {
            const int band_tiles = shape.band * shape.tiles_n;
            const int b = t / band_tiles, r = t - b * band_tiles;
            const int m0 = b * shape.band, width = min(shape.band, shape.tiles_m - m0);
            const int tn = r / width;
            p.expert = 0;
            p.row0 = (m0 + r - tn * width) * BM;
            p.row_end = shape.m;
            p.col0 = tn * BN;
        }
        return p;
    };

    if (warp < 4) {
        if (BN == 256) reg_dealloc<kControlRegs>();
        if (warp == 0 && lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = unit; t < n_tiles && ok; t += n_units) {
                const TilePos p = tile_pos(t);
                const bool small = p.row_end - p.row0 <= kSmallRows;
                const int row_b = p.expert * shape.n + p.col0;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, ctx, 1))) break;
                    const uint32_t dst = s_ring + stage * kStage, bar = bar_full + 8 * stage;
                    mbar_arrive_expect_tx(bar, (uint32_t)((small ? kSmallRows * BK : kABytes) + BN * BK));
                    tma_load_2d(dst + kABytes, &tmap_b, bar, kb * BK, row_b);
                    tma_load_2d(dst, small ? &tmap_a_small : &tmap_a, bar, kb * BK, p.row0);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        if (warp == 1 && lane == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            const uint64_t da0 = make_desc_kmajor_sw128(s_ring), db0 = make_desc_kmajor_sw128(s_ring + kABytes);
            const uint32_t a_hi = (uint32_t)(da0 >> 32), b_hi = (uint32_t)(db0 >> 32);
            bool ok = true;
            for (int t = unit; t < n_tiles && ok; t += n_units) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = mbar_wait(bar_tempty + 8 * acc, acc_phase ^ 1u, ctx, 2))) break;
                    if (!(ok = mbar_wait(bar_full + 8 * stage, phase, ctx, 3))) break;
                    tc_fence_after_sync();
                    const uint32_t a_lo = (uint32_t)da0 + (uint32_t)(stage * (kStage >> 4));
                    const uint32_t b_lo = (uint32_t)db0 + (uint32_t)(stage * (kStage >> 4));
                    const uint32_t d = tmem_base + (uint32_t)(acc * BN);
#pragma unroll
                    for (int i = 0; i < 4; ++i)      // 32 e4m3 along K = 32 bytes = +2 in the encoded address
                        umma_f8_ss(d, a_lo + 2 * i, a_hi, b_lo + 2 * i, b_hi, kIdesc, i != 0 ? 1u : 0u);
                    umma_commit<1>(bar_empty + 8 * stage);
                    umma_commit<1>(bar_tfull + 8 * acc);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
                }
            }
        }
    } else {
        if (BN == 256) reg_alloc<kEpilogueRegs>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t stage_buf = s_epi + (uint32_t)(warp - 4) * kStageBytes;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int t = unit; t < n_tiles && ok; t += n_units) {
            const TilePos p = tile_pos(t);
            const int row = p.row0 + q * 32 + lane;                  // this thread's row
            const int col = p.col0 + half * kCols;                   // this warp's first column
            const float* sa = row < p.row_end ? a_scale + (long long)row * shape.blocks : nullptr;
            const float* sb = col < shape.n ? b_scale + ((long long)p.expert * shape.n_blocks + col / BK) * shape.blocks : nullptr;
            float sum[kCols];
#pragma unroll
            for (int i = 0; i < kCols; ++i) sum[i] = 0.0f;
            float s_next = sa && sb && kb0 < kb1 ? __ldg(sa + kb0) * __ldg(sb + kb0) : 0.0f;
            for (int kb = kb0; kb < kb1; ++kb) {
                const float s = s_next;
                ok = mbar_wait(bar_tfull + 8 * acc, acc_phase, ctx, 4);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after_sync();
                if (sa && sb && kb + 1 < kb1) s_next = __ldg(sa + kb + 1) * __ldg(sb + kb + 1);
                const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * kCols);
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld_32x32b_x32(t_row + c * 32, v);
                    tmem_ld_wait();
                    reg_fence(v);
                    if (c == kCols / 32 - 1) {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        fma2v(sum[c * 32 + i], sum[c * 32 + i + 1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]), s, s,
                              sum[c * 32 + i], sum[c * 32 + i + 1]);
                }
                if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
            }
            if (!ok) break;
            if (split > 1) {
                // One tile a cluster: the ring is drained (every MMA that read it has been waited for
                // through its accumulator), so the partial tile goes there.
                float* part = reinterpret_cast<float*>(smem_gen) + (q * 32 + lane) * kPartPitch + half * kCols;
                if (row < p.row_end) {
#pragma unroll
                    for (int i = 0; i < kCols; i += 4)
                        *reinterpret_cast<float4*>(part + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
                }
                break;
            }
            constexpr int kChunkCols = kChunkBytes / (int)sizeof(OutT);
#pragma unroll
            for (int c = 0; c < kCols / kChunkCols; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (sizeof(OutT) == 4) {
                        w[i] = __float_as_uint(sum[c * kChunkCols + i]);
                    } else {
                        __nv_bfloat162 b2 = __floats2bfloat162_rn(sum[c * kChunkCols + 2 * i], sum[c * kChunkCols + 2 * i + 1]);
                        w[i] = *reinterpret_cast<uint32_t*>(&b2);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    st_shared_v4(stage_buf + (uint32_t)(lane * kChunkBytes + ((j ^ ((lane >> 1) & 3)) << 4)),
                                 w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                __syncwarp();
                const int j = lane & 3, c_out = col + c * kChunkCols + j * (16 / (int)sizeof(OutT));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 8 + (lane >> 2), r_out = p.row0 + q * 32 + r;
                    uint32_t x0, x1, x2, x3;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x0), "=r"(x1), "=r"(x2), "=r"(x3)
                                 : "r"(stage_buf + (uint32_t)(r * kChunkBytes + ((j ^ ((r >> 1) & 3)) << 4))) : "memory");
                    if (r_out < p.row_end && c_out < shape.n)
                        *reinterpret_cast<uint4*>(out + (long long)r_out * shape.n + c_out) = make_uint4(x0, x1, x2, x3);
                }
            }
        }
    }

    __syncwarp();
    tc_fence_before_sync();
    if (split > 1) {
        // Sum of the partial tiles, read through distributed shared memory in the order of K: CTA r of the
        // cluster finishes every split-th vector of the tile.
        cluster_sync_all();
        if (unit < n_tiles) {
            const TilePos p = tile_pos(unit);
            const int rows = min(BM, p.row_end - p.row0), vecs = BN / 4;
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
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem_base, kTmemCols);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
    int64_t experts, m, n, k, tiles;
    int bn, split;
};

// Tile width and split of K.
//   dense: 128 x 256 tiles once they fill the SMs.  With fewer tiles 128-column ones, and where those
//   leave SMs idle the K blocks of a tile are shared by a cluster of up to 8 CTAs (at least two
//   blocks each), which add their partial tiles through distributed shared memory in a fixed order.
//   grouped: the tiles are known on the device only; 256 columns unless N fits 128.
Plan make_plan(const Record& r) {
    Plan p{};
    const bool grouped = r.kernel_id == PB200_K_FP8_GROUPED_GEMM;
    const int64_t* d = r.dims + (grouped ? 1 : 0);
    p.experts = grouped ? r.dims[0] : 0;
    p.m = d[0]; p.n = d[1]; p.k = d[2];
    p.split = 1;
    const int64_t sms = sm_count(), mt = ceil_div(p.m, BM);
    if (grouped) {
        p.bn = p.n > 128 ? 256 : 128;
        // every expert may end in a partial tile
        p.tiles = (mt + p.experts) * ceil_div(p.n, p.bn);
        return p;
    }
    p.bn = mt * ceil_div(p.n, 256) >= sms ? 256 : 128;
    p.tiles = mt * ceil_div(p.n, p.bn);
    if (p.bn == 128) {
        const int64_t blocks = ceil_div(p.k, BK);
        while (p.split < kMaxSplit && p.tiles * p.split * 2 <= sms && blocks >= 4 * p.split) p.split *= 2;
    }
    return p;
}

template <int BN, typename OutT>
int launch_variant(const Record& r, const Plan& p, cudaStream_t stream, void** ptrs, char* err) {
    auto kernel = fp8_gemm_kernel<BN, OutT>;
    static std::atomic<uint64_t> attr_set{0};   // bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(attr_set.load(std::memory_order_relaxed) & (1ull << (dev & 63)))) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemTotal);
        if (e != cudaSuccess) { set_err(err, "cudaFuncSetAttribute(smem=%d): %s", kSmemTotal, cudaGetErrorString(e)); return PB200_ERR_LAUNCH; }
        attr_set.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
    auto map = [&](CUtensorMap* m, const void* base, int64_t rows, uint32_t box_rows) {
        uint64_t dims[2] = {(uint64_t)p.k, (uint64_t)rows};
        uint64_t str[1] = {(uint64_t)p.k};
        uint32_t box[2] = {BK, box_rows};
        return make_tensor_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, err);
    };
    CUtensorMap ta, ta_small, tb;
    if (int rc = map(&ta, ptrs[0], p.m, BM)) return rc;
    if (int rc = map(&ta_small, ptrs[0], p.m, kSmallRows)) return rc;
    if (int rc = map(&tb, ptrs[2], p.n * (p.experts ? p.experts : 1), BN)) return rc;
    Shape s;
    s.m = (int)p.m;
    s.n = (int)p.n;
    s.blocks = (int)ceil_div(p.k, BK);
    s.tiles_m = (int)ceil_div(p.m, BM);
    s.tiles_n = (int)ceil_div(p.n, BN);
    s.band = s.tiles_m < 16 ? s.tiles_m : 16;
    s.experts = (int)p.experts;
    s.n_blocks = (int)ceil_div(p.n, BK);
    s.split = p.split;
    const int64_t sms = sm_count();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.split > 1 ? p.tiles * p.split : p.tiles < sms ? p.tiles : sms));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemTotal;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.split > 1 ? 2 : 1;
    const bool grouped = p.experts > 0;
    const int* offsets = grouped ? (const int*)ptrs[4] : nullptr;
    OutT* out = (OutT*)ptrs[grouped ? 5 : 4];
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ta, ta_small, tb, (const float*)ptrs[1], (const float*)ptrs[3], offsets, out, s,
                                       device_status_ptr(), (int)r.kernel_id);
    if (e != cudaSuccess) {
        set_err(err, "fp8 gemm launch failed (BN=%d split=%d): %s", BN, p.split, cudaGetErrorString(e));
        return p.split > 1 ? PB200_ERR_CLUSTER : PB200_ERR_LAUNCH;
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
    if (p.m + BM > 0x7fffffffLL || (grouped ? p.experts : 1) * p.n + 256 > 0x7fffffffLL || p.k + BK > 0x7fffffffLL ||
        p.tiles > 0x3fffffffLL) {
        set_err(err, "extent exceeds 2^31-1");
        return PB200_ERR_BAD_SHAPE;
    }
    pb200_geometry& g = r.geom;
    const int64_t sms = sm_count();
    g.grid[0] = (uint32_t)(p.split > 1 ? p.tiles * p.split : p.tiles < sms ? p.tiles : sms);
    g.grid[1] = g.grid[2] = 1;
    g.block[0] = kThreads;
    g.block[1] = g.block[2] = 1;
    g.cluster[0] = (uint32_t)p.split;
    g.cluster[1] = g.cluster[2] = 1;
    g.smem_bytes = kSmemTotal;
    g.n_inputs = grouped ? 5 : 4;
    g.n_outputs = 1;
    return PB200_OK;
}

int launch_fp8_gemm(const Record& r, cudaStream_t stream, void** ptrs, char* err) {
    const Plan p = make_plan(r);
    const bool b16 = (r.flags & PB200_F_OUT_BF16) != 0;
    if (p.bn == 256)
        return b16 ? launch_variant<256, __nv_bfloat16>(r, p, stream, ptrs, err) : launch_variant<256, float>(r, p, stream, ptrs, err);
    return b16 ? launch_variant<128, __nv_bfloat16>(r, p, stream, ptrs, err) : launch_variant<128, float>(r, p, stream, ptrs, err);
}

}  // namespace pb200
