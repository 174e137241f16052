// Block-scaled e4m3 GEMM for a few rows of A (single tokens, small batches of them):
//   D[m,n] = sum over 128-wide blocks b of K of
//            a_scale[m,b] * b_scale[n/128,b] * sum_{k in b} A[m,k] * B_T[n,k]
//
// The product reads the weight once and does next to nothing with it, so this is a stream with the
// shortest possible way in and out: a warp takes 16 weight rows x one scale block at a time straight
// from memory into registers (four 16-byte loads a lane; the loads of DEPTH blocks are in flight),
// the warps of a CTA take the scale blocks in turn and add their f32 sums through shared memory in the
// order of the warps.  No barriers to set up, no TMEM, no clusters: that is what a call of a few
// microseconds pays for in the tiled kernel (fp8_gemm_sm100.cu).
//
// Arithmetic: e4m3 -> f16 is exact, and mma.sync m16n8k16 adds the exact products of one scale block in
// f32, with the weight as the 16-row operand and eight tokens as the columns.  (mma.sync on e4m3 operands
// is emulated on sm_100 and measured 1.7 times slower.)  Both operands are fetched 16 bytes a lane: lane
// (g, t) holds k = 16 t .. 16 t + 15 of its row in a 64-wide half block, and the instruction's k index is
// taken as that permutation of k on both sides.
#include "common.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

namespace pb200 {
namespace {

constexpr int kRows = 16;                    // weight rows of a CTA
constexpr int kBlock = 128;                  // scale block
constexpr int kMaxWarps = 16;
constexpr int kAhead = 2048;                 // bytes of a weight row asked for ahead of the previous kernel's end

struct SkinnyArgs {
    const uint8_t* a;
    const float* a_scale;
    const uint8_t* b;
    const float* b_scale;
    void* out;
    int m, n, k;
    int blocks;               // scale blocks of K
};

__device__ __forceinline__ uint4 ld_weight(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// Four e4m3 -> two f16x2, exact (NaN stays NaN).
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void widen16(const uint4& v, uint32_t (&h)[8]) {
    widen(v.x, h[0], h[1]);
    widen(v.y, h[2], h[3]);
    widen(v.z, h[4], h[5]);
    widen(v.w, h[6], h[7]);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// MT: tiles of eight tokens.
template <int MT, int DEPTH, typename OutT>
__global__ void __launch_bounds__(kMaxWarps * 32) fp8_skinny_kernel(SkinnyArgs p) {
    extern __shared__ float part[];                       // [warps][8 * MT][kRows]
    constexpr int kTok = 8 * MT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kRows;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint8_t* w_row[2];                              // rows g and g + 8
    bool w_there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w_there[i] = n0 + g + 8 * i < p.n;
        w_row[i] = p.b + (long long)(w_there[i] ? n0 + g + 8 * i : 0) * p.k + 16 * t;
    }
    ptx::pdl_launch_dependents();
    // CTAs that start while the previous kernel runs bring the beginning of their weight rows into L2 meanwhile
    // (whatever the previous kernel still writes there is seen all the same: L2 is where writes arrive, and the
    // loads below come after the wait).  Back to back from HBM 1 x 4096 x 4096 takes 4.9 us instead of 5.4 and
    // 1 x 8192 x 8192 14.7 instead of 15.4; whole rows would give the first 0.15 us less and the second 2 more,
    // and a weight that lies in L2 already pays 0.3 and 1.6 us for being asked for twice.
    if (threadIdx.x < kRows && n0 + (int)threadIdx.x < p.n)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                     :: "l"(p.b + (long long)(n0 + (int)threadIdx.x) * p.k), "r"(min(p.k, kAhead)) : "memory");
    ptx::pdl_wait();

    const float* sb = p.b_scale + (long long)(n0 / kBlock) * p.blocks;
    const uint8_t* x_row[MT];
    bool x_there[MT];
    const float* sa[MT][2];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        x_there[j] = 8 * j + g < p.m;
        x_row[j] = p.a + (long long)(x_there[j] ? 8 * j + g : 0) * p.k + 16 * t;
#pragma unroll
        for (int i = 0; i < 2; ++i) sa[j][i] = p.a_scale + (long long)min(8 * j + 2 * t + i, p.m - 1) * p.blocks;
    }
    float acc[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;

    uint4 w[DEPTH][2][2], x[DEPTH][2][MT];                // [64-column half][row]
    float s[DEPTH][MT][2], s_b[DEPTH];
    auto load = [&](int d, int b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = b * kBlock + 64 * h;
            const bool in = k + 16 * t < p.k;
#pragma unroll
            for (int i = 0; i < 2; ++i) w[d][h][i] = w_there[i] && in ? ld_weight(w_row[i] + k) : zero;
#pragma unroll
            for (int j = 0; j < MT; ++j) x[d][h][j] = x_there[j] && in ? __ldg(reinterpret_cast<const uint4*>(x_row[j] + k)) : zero;
        }
        s_b[d] = __ldg(sb + b);
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) s[d][j][i] = __ldg(sa[j][i] + b);
    };
    auto use = [&](int d) {
        float c[MT][4];
#pragma unroll
        for (int j = 0; j < MT; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t lo[8], hi[8];                        // rows g, g + 8
            widen16(w[d][h][0], lo);
            widen16(w[d][h][1], hi);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                uint32_t tok[8];
                widen16(x[d][h][j], tok);
#pragma unroll
                for (int q = 0; q < 4; ++q) mma_f16(c[j], lo[2 * q], hi[2 * q], lo[2 * q + 1], hi[2 * q + 1], tok[2 * q], tok[2 * q + 1]);
            }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const float s0 = s[d][j][0] * s_b[d], s1 = s[d][j][1] * s_b[d];
            acc[j][0] = fmaf(c[j][0], s0, acc[j][0]);
            acc[j][1] = fmaf(c[j][1], s1, acc[j][1]);
            acc[j][2] = fmaf(c[j][2], s0, acc[j][2]);
            acc[j][3] = fmaf(c[j][3], s1, acc[j][3]);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (warp + d * n_warps < p.blocks) load(d, warp + d * n_warps);
    for (int b0 = warp; b0 < p.blocks; b0 += DEPTH * n_warps) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int b = b0 + d * n_warps;
            if (b >= p.blocks) break;
            use(d);
            if (b + DEPTH * n_warps < p.blocks) load(d, b + DEPTH * n_warps);
        }
    }
    // [token][row], so that the sums below read and write consecutive rows
    float* mine = part + warp * (kTok * kRows);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int tok = 8 * j + 2 * t;
        mine[tok * kRows + g] = acc[j][0];
        mine[(tok + 1) * kRows + g] = acc[j][1];
        mine[tok * kRows + g + 8] = acc[j][2];
        mine[(tok + 1) * kRows + g + 8] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(kTok, p.m) * kRows; i += blockDim.x) {
        float sum = 0.0f;
        for (int v = 0; v < n_warps; ++v) sum += part[v * (kTok * kRows) + i];
        const int tok = i / kRows, row = i - tok * kRows;
        if (n0 + row < p.n) store_value(reinterpret_cast<OutT*>(p.out) + (long long)tok * p.n + n0 + row, sum);
    }
}

}  // namespace

// Warps of a CTA, which share K: enough of them in all to fill the SMs (16 an SM), at most one for each
// scale block.
int fp8_skinny_warps(int64_t n, int64_t k) {
    const int64_t blocks = (k + kBlock - 1) / kBlock, ctas = fp8_skinny_grid(n), want = (int64_t)sm_count() * 16;
    int64_t warps = 4;
    while (warps < kMaxWarps && ctas * warps * 2 <= want) warps *= 2;
    return (int)(blocks < warps ? blocks : warps);
}
int64_t fp8_skinny_grid(int64_t n) { return (n + kRows - 1) / kRows; }
static int token_tiles_of(int64_t m) { return m <= 8 ? 1 : m <= 16 ? 2 : 4; }
size_t fp8_skinny_smem(int64_t m, int64_t n, int64_t k) {
    return (size_t)fp8_skinny_warps(n, k) * kRows * 8 * token_tiles_of(m) * sizeof(float);
}

int launch_fp8_skinny(const Record& r, int64_t m, int64_t n, int64_t k, cudaStream_t stream, void** ptrs, char* err) {
    SkinnyArgs a;
    a.a = (const uint8_t*)ptrs[0];
    a.a_scale = (const float*)ptrs[1];
    a.b = (const uint8_t*)ptrs[2];
    a.b_scale = (const float*)ptrs[3];
    a.out = ptrs[4];
    a.m = (int)m; a.n = (int)n; a.k = (int)k;
    a.blocks = (int)((k + kBlock - 1) / kBlock);
    const int token_tiles = token_tiles_of(m);
    const size_t smem = fp8_skinny_smem(m, n, k);
    const dim3 grid((unsigned)fp8_skinny_grid(n)), block(32 * fp8_skinny_warps(n, k));
    const bool b16 = (r.flags & PB200_F_OUT_BF16) != 0;
    cudaError_t e;
    if (token_tiles == 1)
        e = b16 ? launch_with_pdl(fp8_skinny_kernel<1, 3, __nv_bfloat16>, grid, block, smem, stream, a)
                : launch_with_pdl(fp8_skinny_kernel<1, 3, float>, grid, block, smem, stream, a);
    else if (token_tiles == 2)
        e = b16 ? launch_with_pdl(fp8_skinny_kernel<2, 2, __nv_bfloat16>, grid, block, smem, stream, a)
                : launch_with_pdl(fp8_skinny_kernel<2, 2, float>, grid, block, smem, stream, a);
    else                          // one block a warp (make_plan): no depth, which would not fit the registers
        e = b16 ? launch_with_pdl(fp8_skinny_kernel<4, 1, __nv_bfloat16>, grid, block, smem, stream, a)
                : launch_with_pdl(fp8_skinny_kernel<4, 1, float>, grid, block, smem, stream, a);
    if (e != cudaSuccess) { set_err(err, "fp8 gemm launch failed (few rows): %s", cudaGetErrorString(e)); return PB200_ERR_LAUNCH; }
    return PB200_OK;
}

}  // namespace pb200
