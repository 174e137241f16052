// Mixture-of-experts token movement for sm_100a, around the grouped GEMMs:
//   route      expert ids -> a stable sort of the T*k entries by expert (both directions of the map
//              and the experts' row offsets, padded to the grouped kernels' row blocks)
//   dispatch   tokens -> rows sorted by expert (rows as they are, or quantised to e4m3 with a scale
//              for each 128 columns), and its gradient
//   combine    rows -> tokens, weighted, and its gradient
// and the quantisation of plain matrices that the 8-bit GEMM takes.
//
// Everything but the sort moves bytes and computes next to nothing, so those kernels are bound by
// HBM: 16-byte accesses, consecutive lanes on consecutive segments, every independent load issued
// before the first use, each input read once and each output written once.  No atomics: every sum
// has a fixed order, so results are the same from run to run.  Measured at 8192 tokens x 4 choices over 32
// experts, 4096 columns, bf16, rows padded to 128 (algorithmic bytes over time, inputs larger than L2):
// dispatch 6.35 TB/s, dispatch into e4m3 6.25, its gradient 6.6, combine 6.55, its gradient 6.46; a plain
// copy reaches 6.54.
#include "common.cuh"
#include "ptx.cuh"

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace pb200 {
namespace {

constexpr int kThreads = 128;                 // movement kernels: 4 warps, one unit of work per warp
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTopK = 32;                  // one lane holds one choice's row and weight
constexpr int kMaxExperts = 1024;
constexpr int kMaxBlock = 1024;
constexpr int kScaleBlock = 128;
constexpr int64_t kMaxExtent = 0x7fff0000;    // rows and columns; 65535 more fit 32 bits (a whole grid's step past the last need not)

__device__ __forceinline__ void pdl_prologue() {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
}

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void st_stream(uint4* p, const uint4& v) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};"
                 :: "l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A 16-byte vector as f32 values: 8 bf16 or 4 f32.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// ---------------------------------------------------------------------------
// Route: a stable counting sort in one launch of one cluster (up to 32768 entries; see below for more).
//
// Entry i = t*k + j asks for expert ids[i].  CTA c of the cluster owns a contiguous range of
// entries and each of its warps a contiguous part of that, so "earlier entry" is "earlier step of
// the same warp, or an earlier warp, or an earlier CTA".  A warp walks its part 32 entries at a
// time; ballots give each lane its rank among the lanes with the same expert, and the warp's
// running counters in shared memory the rest.  Counters are then prefix-summed over warps (each
// thread one expert), over CTAs (through distributed shared memory) and, padded to `block` rows,
// over experts; the row of an entry is the sum of the three.  Rows that no entry owns get entry -1
// in the same launch, so nothing has to be cleared beforehand.
//
// Latency-bound: the ids are read once (4 or 8 bytes an entry), the maps written once.  In a chain of
// graph launches 128 entries take 3.2 us, 32768 (eight CTAs, 32 experts) 6.5 us.
// ---------------------------------------------------------------------------
constexpr int kRouteThreads = 1024;           // of a CTA; kRouteFewThreads for few entries and experts
constexpr int kRouteFewThreads = 256;
constexpr int kRouteFewEntries = 256, kRouteFewExperts = 128;
constexpr int kRouteMaxCtas = 8;
constexpr int kMaxIdBits = 10;                // ids below kMaxExperts
static_assert(1 << kMaxIdBits >= kMaxExperts, "id bits");
constexpr int kRouteRegSteps = 4;            // steps of a warp, whose ids and ranks stay in registers
constexpr int64_t kRouteClusterEntries = (int64_t)kRouteMaxCtas * kRouteThreads * kRouteRegSteps;      // more take two launches
static_assert(kRouteFewEntries <= kRouteFewThreads * kRouteRegSteps, "few entries stay in registers");
static_assert(kRouteFewExperts <= kRouteFewThreads, "a thread for each expert");

struct RouteArgs {
    const void* ids;
    int* row_of;
    int* entry_of;
    int* offsets;
    int n;                // entries
    int experts;
    int block;
    int rows;
    int per_warp;         // entries of a warp, a multiple of 32
};

template <typename IdT>
__device__ __forceinline__ int load_id(const void* ids, int i, int n, int experts) {
    if (i >= n) return -1;
    const IdT v = __ldg(reinterpret_cast<const IdT*>(ids) + i);
    return v >= 0 && v < (IdT)experts ? (int)v : -1;      // ids outside [0, experts) are dropped
}

// Rank of this lane's entry among the entries of its expert that this warp has seen; advances the counter.
// The lanes with the same expert are found with one ballot for each bit of the id (cheaper than
// match_any, which takes one step for each distinct value).
__device__ __forceinline__ int warp_rank(int* counters, int id, int lane, int id_bits) {
    unsigned same = __ballot_sync(0xffffffffu, id >= 0);
    if (id < 0) same = ~same;
#pragma unroll
    for (int b = 0; b < kMaxIdBits; ++b) {
        if (b >= id_bits) break;
        const bool bit = (id >> b) & 1;
        const unsigned votes = __ballot_sync(0xffffffffu, bit);
        same &= bit ? votes : ~votes;
    }
    const unsigned before = same & ((1u << lane) - 1u);
    int base = 0;
    if (id >= 0) base = counters[id];
    __syncwarp();
    if (id >= 0 && before == 0) counters[id] = base + __popc(same);
    __syncwarp();
    return base + __popc(before);
}

template <typename IdT, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) route_kernel(RouteArgs a) {
    constexpr int kWarpsHere = THREADS / 32;
    pdl_prologue();
    extern __shared__ int smem[];
    const int E = a.experts;
    int* counters = smem;                           // [warps][E]: counts, then prefix over warps
    int* cta_count = counters + kWarpsHere * E;    // [E], read by the other CTAs
    int* base = cta_count + E;                      // [E] first row of this CTA's entries of an expert
    int* filled = base + E;                         // [E] end of the expert's entries (row)
    int* ends = filled + E;                         // [E] end of the expert's rows
    int* local = ends + E;                          // [E] first place of an expert among this CTA's sorted entries
    int2* sorted = reinterpret_cast<int2*>(local + E + (E & 1));      // (row, entry) of this CTA's entries, by expert
    __shared__ int warp_total[32], warp_own[32];

    uint32_t n_ctas;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n_ctas));
    const int rank = (int)ptx::cluster_ctarank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int id_bits = 32 - __clz(E - 1);          // E = 1: none
    const int first = (rank * kWarpsHere + warp) * a.per_warp;
    const int steps = first < a.n ? (min(a.per_warp, a.n - first) + 31) / 32 : 0;

    int my_id[kRouteRegSteps], my_rank[kRouteRegSteps];
#pragma unroll
    for (int r = 0; r < kRouteRegSteps; ++r) my_id[r] = r < steps ? load_id<IdT>(a.ids, first + r * 32 + lane, a.n, E) : -1;
    for (int i = tid; i < kWarpsHere * E; i += THREADS) counters[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRouteRegSteps; ++r)
        if (r < steps) my_rank[r] = warp_rank(counters + warp * E, my_id[r], lane, id_bits);
    __syncthreads();
    // prefix over warps: counters[w][e] = entries of e in earlier warps of this CTA
    for (int e = tid; e < E; e += THREADS) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < kWarpsHere; ++w) {
            const int c = counters[w * E + e];
            counters[w * E + e] = run;
            run += c;
        }
        cta_count[e] = run;
    }
    if (n_ctas > 1) ptx::cluster_sync_all(); else __syncthreads();
    // totals over CTAs, then a block-wide exclusive prefix of the padded totals (E <= THREADS)
    int total = 0, before = 0, own_count = 0;
    if (tid < E) {
        own_count = cta_count[tid];
        const uint32_t own = ptx::smem_u32(cta_count + tid);
        int v[kRouteMaxCtas];
#pragma unroll
        for (int c = 0; c < kRouteMaxCtas; ++c) {        // all reads in flight at once
            v[c] = 0;
            if (c < (int)n_ctas)
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[c]) : "r"(ptx::map_to_cta(own, (uint32_t)c)) : "memory");
        }
#pragma unroll
        for (int c = 0; c < kRouteMaxCtas; ++c) {
            if (c < rank) before += v[c];
            total += v[c];
        }
    }
    __syncwarp();
    if (n_ctas > 1) ptx::cluster_arrive();          // this warp has read the others' counts
    const int padded = (total + a.block - 1) / a.block * a.block;
    int incl = padded, own = own_count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o), u = __shfl_up_sync(0xffffffffu, own, o);
        if (lane >= o) { incl += v; own += u; }
    }
    if (lane == 31) { warp_total[warp] = incl; warp_own[warp] = own; }
    __syncthreads();
    if (warp < 2) {
        int* totals = warp == 0 ? warp_total : warp_own;
        int v = lane < kWarpsHere ? totals[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        totals[lane] = v;
    }
    __syncthreads();
    const int end = incl + (warp > 0 ? warp_total[warp - 1] : 0);
    if (tid < E) {
        local[tid] = own - own_count + (warp > 0 ? warp_own[warp - 1] : 0);
        const int start = end - padded;
        base[tid] = start + before;
        filled[tid] = start + total;
        ends[tid] = end;
        if (rank == 0) {
            a.offsets[tid + 1] = min(end, a.rows);
            if (tid == 0) a.offsets[0] = 0;
        }
    }
    __syncthreads();
    // Entries go to entry_of by way of shared memory, sorted, so that neighbouring lanes store neighbouring
    // rows (stored straight from the lanes they cost a sector each, and eight SMs store one a clock).
#pragma unroll
    for (int r = 0; r < kRouteRegSteps; ++r) {
        const int i = first + r * 32 + lane, id = my_id[r];
        if (r < steps && i < a.n) {
            int row = -1;
            if (id >= 0) {
                const int k = counters[warp * E + id] + my_rank[r];
                row = base[id] + k;
                if (row >= a.rows) row = -1;                        // no room: dropped
                sorted[local[id] + k] = make_int2(row, i);
            }
            a.row_of[i] = row;
        }
    }
    __syncthreads();
    for (int k = tid; k < warp_own[kWarpsHere - 1]; k += THREADS) {
        const int2 at = sorted[k];
        if (at.x >= 0) a.entry_of[at.x] = at.y;
    }
    // rows without an entry: each expert's padding, then everything behind the last expert
    for (int e = rank * kWarpsHere + warp; e < E; e += (int)n_ctas * kWarpsHere)
        for (int r = filled[e] + lane; r < min(ends[e], a.rows); r += 32) a.entry_of[r] = -1;
    static_assert(kMaxExtent + kRouteMaxCtas * kRouteThreads <= 0x7fffffff, "a cluster's step past the last row fits 32 bits");
    for (int r = ends[E - 1] + rank * THREADS + tid; r < a.rows; r += (int)n_ctas * THREADS) a.entry_of[r] = -1;
    if (n_ctas > 1) ptx::cluster_wait();            // shared memory must outlive the other CTAs' reads
}

// The same sort for more entries than a cluster's registers hold, on all SMs in two launches.  The first
// ranks: row_of takes an entry's rank among its expert's entries of this CTA, counts[e][c] their number.  The
// second adds what earlier CTAs and experts have (a warp sums an expert's counts, lanes along the CTAs) and places.
// 65536 entries over 32 experts 6.5 us (on one cluster of eight CTAs 10.1), 524288 over 256 19 (96); at 32768 the
// cluster is as quick (6.5 against 6.9 over 32 experts, 8.2 against 8.9 over 256) and takes one launch.
template <typename IdT>
__global__ void __launch_bounds__(kRouteThreads, 1) route_rank_kernel(RouteArgs a, int* counts) {
    pdl_prologue();
    extern __shared__ int counters[];               // [warps][E]: counts, then prefix over warps
    constexpr int kWarpsHere = kRouteThreads / 32;
    const int E = a.experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int id_bits = 32 - __clz(E - 1);
    const int first = ((int)blockIdx.x * kWarpsHere + warp) * a.per_warp;
    const int steps = first < a.n ? (min(a.per_warp, a.n - first) + 31) / 32 : 0;
    for (int i = tid; i < kWarpsHere * E; i += kRouteThreads) counters[i] = 0;
    __syncthreads();
    int next = load_id<IdT>(a.ids, first + lane, steps > 0 ? a.n : 0, E);
    for (int r = 0; r < steps; ++r) {
        const int i = first + r * 32 + lane, id = next;
        next = r + 1 < steps ? load_id<IdT>(a.ids, i + 32, a.n, E) : -1;
        const int rk = warp_rank(counters + warp * E, id, lane, id_bits);
        if (i < a.n) a.row_of[i] = rk;              // kept for the pass below of this same thread
    }
    __syncthreads();
    for (int e = tid; e < E; e += kRouteThreads) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < kWarpsHere; ++w) {
            const int c = counters[w * E + e];
            counters[w * E + e] = run;
            run += c;
        }
        counts[e * gridDim.x + blockIdx.x] = run;
    }
    __syncthreads();
#pragma unroll 4
    for (int r = 0; r < steps; ++r) {
        const int i = first + r * 32 + lane, id = load_id<IdT>(a.ids, i, a.n, E);
        if (id >= 0) a.row_of[i] += counters[warp * E + id];
    }
}

template <typename IdT>
__global__ void __launch_bounds__(kRouteThreads, 1) route_place_kernel(RouteArgs a, const int* counts) {
    pdl_prologue();
    __shared__ int base[kMaxExperts];               // first row of this CTA's entries of an expert
    __shared__ int filled[kMaxExperts];             // the expert's entries, then the end of its entries (row)
    __shared__ int ends[kMaxExperts];               // end of the expert's rows
    __shared__ int warp_total[32];
    constexpr int kWarpsHere = kRouteThreads / 32;
    const int E = a.experts, ctas = (int)gridDim.x, rank = (int)blockIdx.x;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kGroup = 8;                       // experts whose loads are in flight together
    for (int e0 = warp; e0 < E; e0 += kGroup * kWarpsHere) {
        int before[kGroup] = {}, total[kGroup] = {};
#pragma unroll 2
        for (int c = lane; c < ctas; c += 32) {
            int v[kGroup];
#pragma unroll
            for (int g = 0; g < kGroup; ++g) v[g] = e0 + g * kWarpsHere < E ? counts[(e0 + g * kWarpsHere) * ctas + c] : 0;
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
                total[g] += v[g];
                if (c < rank) before[g] += v[g];
            }
        }
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            if (e0 + g * kWarpsHere >= E) break;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                before[g] += __shfl_xor_sync(0xffffffffu, before[g], o);
                total[g] += __shfl_xor_sync(0xffffffffu, total[g], o);
            }
            if (lane == 0) { base[e0 + g * kWarpsHere] = before[g]; filled[e0 + g * kWarpsHere] = total[g]; }
        }
    }
    __syncthreads();
    const int total = tid < E ? filled[tid] : 0, padded = (total + a.block - 1) / a.block * a.block;
    int end = padded;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
    }
    if (lane == 31) warp_total[warp] = end;
    __syncthreads();
    if (warp == 0) {
        int v = warp_total[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        warp_total[lane] = v;
    }
    __syncthreads();
    if (warp > 0) end += warp_total[warp - 1];
    if (tid < E) {
        base[tid] += end - padded;
        filled[tid] = end - padded + total;
        ends[tid] = end;
        if (rank == 0) {
            a.offsets[tid + 1] = min(end, a.rows);
            if (tid == 0) a.offsets[0] = 0;
        }
    }
    __syncthreads();
    const int first = (rank * kWarpsHere + warp) * a.per_warp;
    const int steps = first < a.n ? (min(a.per_warp, a.n - first) + 31) / 32 : 0;
#pragma unroll 4
    for (int r = 0; r < steps; ++r) {
        const int i = first + r * 32 + lane, id = load_id<IdT>(a.ids, i, a.n, E);
        if (i >= a.n) continue;
        int row = -1;
        if (id >= 0) {
            row = base[id] + a.row_of[i];
            if (row < a.rows) a.entry_of[row] = i; else row = -1;
        }
        a.row_of[i] = row;
    }
    // rows without an entry, as above
    for (int e = rank * kWarpsHere + warp; e < E; e += ctas * kWarpsHere)
        for (int r = filled[e] + lane; r < min(ends[e], a.rows); r += 32) a.entry_of[r] = -1;
    for (int64_t r = ends[E - 1] + rank * kRouteThreads + tid; r < a.rows; r += ctas * kRouteThreads) a.entry_of[r] = -1;
}

// ---------------------------------------------------------------------------
// Zero rows.  A unit is 32 rows x one segment: a lane looks at one row, the warp then clears its
// segment of every row that no entry owns.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void zero_unowned(uint4* out, const int* __restrict__ entry_of, int64_t row0, int rows, int vecs,
                                             int vec0, int vec1, int lane) {
    const int64_t r = row0 + lane;
    unsigned todo = __ballot_sync(0xffffffffu, r < rows && __ldg(entry_of + r) < 0);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    while (todo) {
        const int b = __ffs(todo) - 1;
        todo &= todo - 1;
        uint4* dst = out + (row0 + b) * vecs;
        for (int v = vec0 + lane; v < vec1; v += 32) st_stream(dst + v, zero);
    }
}

// ---------------------------------------------------------------------------
// Dispatch: a warp reads U x 512 bytes of one token once and writes them to its k rows.  In token
// order the tokens are read once from HBM; in row order they would be read k times.
// ---------------------------------------------------------------------------
struct MoveArgs {
    const void* src;              // tokens (dispatch) or rows (combine)
    const int* row_of;
    const int* entry_of;
    const float* weights;
    void* dst;
    float* dst_scale;
    const void* grad;
    void* d_rows;
    float* d_weights;
    int64_t tokens;
    int64_t zero_units;           // units before the tokens' ones
    int top_k;
    int rows;
    int vecs;                     // 16-byte vectors of a row
    int segs;                     // segments of a row
    int width;                    // columns
    int scale_cols;
};

template <int U>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(MoveArgs a) {
    pdl_prologue();
    const int lane = threadIdx.x & 31;
    int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    uint4* out = reinterpret_cast<uint4*>(a.dst);
    if (unit < a.zero_units) {
        const int seg = (int)(unit % a.segs);
        zero_unowned(out, a.entry_of, unit / a.segs * 32, a.rows, a.vecs, seg * 32 * U, min(a.vecs, (seg + 1) * 32 * U), lane);
        return;
    }
    unit -= a.zero_units;
    const int64_t t = unit / a.segs;
    if (t >= a.tokens) return;
    const int v0 = (int)(unit - t * a.segs) * 32 * U + lane;
    const uint4* x = reinterpret_cast<const uint4*>(a.src) + t * a.vecs;
    const int my_row = lane < a.top_k ? __ldg(a.row_of + t * a.top_k + lane) : -1;
    uint4 d[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (v0 + 32 * u < a.vecs) d[u] = ld_stream(x + v0 + 32 * u);
    for (int j = 0; j < a.top_k; ++j) {
        const int r = __shfl_sync(0xffffffffu, my_row, j);
        if (r < 0 || r >= a.rows) continue;
        uint4* dst = out + (int64_t)r * a.vecs;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v0 + 32 * u < a.vecs) st_stream(dst + v0 + 32 * u, d[u]);
    }
}

// ---------------------------------------------------------------------------
// (Quantising 8192 x 8192 bf16 takes 33.2 us = 6.1 TB/s; two steps a warp instead of four 36.9, eight 38.9.)
// Quantisation of 128-column blocks: s = max(amax / 448, 2^-120), q = e4m3(x * (1 / s)), in f32 with
// every step rounded to nearest.  2^-120 keeps 1/s finite, so that an all-zero block gives zeros.
// amax ignores NaN: a NaN stays in its own element; an infinity makes its block's products NaN.
// A lane holds 8 columns, 16 lanes a block, a warp two blocks.
// ---------------------------------------------------------------------------
constexpr float kFp8Max = 448.0f;

__device__ __forceinline__ float block_scale(float amax) {
    return fmaxf(__fdiv_rn(amax, kFp8Max), 0x1p-120f);
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float inv) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
// 8 consecutive columns; columns come in multiples of 16, so 8 of them are all there or not at all.
template <typename T> __device__ __forceinline__ void load8(const T* p, bool there, float (&v)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, bool there, float (&v)[8]) {
    Vec<__nv_bfloat16>::unpack(there ? ld_stream(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0), v);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, bool there, float (&v)[8]) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    const uint4 lo = there ? ld_stream(reinterpret_cast<const uint4*>(p)) : z;
    const uint4 hi = there ? ld_stream(reinterpret_cast<const uint4*>(p) + 1) : z;
    float a[4], b[4];
    Vec<float>::unpack(lo, a);
    Vec<float>::unpack(hi, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}
__device__ __forceinline__ float amax_of_16_lanes(float m) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Rows quantised for each 1 x 128 block.  ROUTED: token t goes to its k rows, and rows that no entry
// owns become zeros with scale 0; otherwise row t goes to row t.  A warp takes U x 256 columns.
template <typename T, int U, bool ROUTED>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(MoveArgs a) {
    pdl_prologue();
    const int lane = threadIdx.x & 31;
    int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    uint8_t* q_out = reinterpret_cast<uint8_t*>(a.dst);
    if (ROUTED) {
        if (unit < a.zero_units) {
            const int seg = (int)(unit % a.segs);
            const int64_t row0 = unit / a.segs * 32;
            zero_unowned(reinterpret_cast<uint4*>(q_out), a.entry_of, row0, a.rows, a.vecs, seg * 16 * U,
                         min(a.vecs, (seg + 1) * 16 * U), lane);
            const int64_t r = row0 + lane;
            if (r < a.rows && __ldg(a.entry_of + r) < 0)
                for (int c = seg * 2 * U; c < min(a.scale_cols, (seg + 1) * 2 * U); ++c) a.dst_scale[r * a.scale_cols + c] = 0.0f;
            return;
        }
        unit -= a.zero_units;
    }
    const int64_t t = unit / a.segs;
    if (t >= a.tokens) return;
    const int c0 = (int)(unit - t * a.segs) * 256 * U + lane * 8;
    const T* x = reinterpret_cast<const T*>(a.src) + t * a.width;
    int my_row = -1;
    if (ROUTED && lane < a.top_k) my_row = __ldg(a.row_of + t * a.top_k + lane);
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) load8<T>(x + c0 + 256 * u, c0 + 256 * u < a.width, v[u]);
    uint2 q[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        scale[u] = block_scale(amax_of_16_lanes(amax8(v[u])));
        q[u] = quantize8(v[u], __frcp_rn(scale[u]));
    }
    // lane i of the first 2 U holds the scale of the segment's block i, so that they leave in one store
    float my_scale = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float v = __shfl_sync(0xffffffffu, scale[u], (lane & 1) * 16);
        if (lane >> 1 == u) my_scale = v;
    }
    const int scale_col = (c0 - lane * 8) / kScaleBlock + lane;
    const int n_dst = ROUTED ? a.top_k : 1;
    for (int j = 0; j < n_dst; ++j) {
        const int64_t r = ROUTED ? (int64_t)__shfl_sync(0xffffffffu, my_row, j) : t;
        if (ROUTED && (r < 0 || r >= a.rows)) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + 256 * u;
            if (c < a.width) __stcs(reinterpret_cast<uint2*>(q_out + r * a.width + c), q[u]);
        }
        if (lane < 2 * U && scale_col < a.scale_cols) a.dst_scale[r * a.scale_cols + scale_col] = my_scale;
    }
}

// 128 x 128 blocks (weights): a CTA of 512 threads holds one block, 4 rows x 8 columns a thread.
constexpr int kBlockThreads = 512;
constexpr int kBlockSteps = kScaleBlock * kScaleBlock / (8 * kBlockThreads);
constexpr int kBlockStep = kScaleBlock / kBlockSteps;          // rows between a thread's
template <typename T>
__global__ void __launch_bounds__(kBlockThreads) quantize_blocks_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                        float* __restrict__ scales, int64_t rows, int cols,
                                                                        int scale_cols) {
    pdl_prologue();
    __shared__ float part[kBlockThreads / 32];
    const int64_t row0 = (int64_t)(blockIdx.x / scale_cols) * kScaleBlock + threadIdx.x / 16;
    const int col = (int)(blockIdx.x % scale_cols) * kScaleBlock + (threadIdx.x % 16) * 8;
    float v[kBlockSteps][8];
#pragma unroll
    for (int i = 0; i < kBlockSteps; ++i)
        load8<T>(x + (row0 + kBlockStep * i) * cols + col, row0 + kBlockStep * i < rows && col < cols, v[i]);
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlockSteps; ++i) m = fmaxf(m, amax8(v[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (int i = 1; i < kBlockThreads / 32; ++i) m = fmaxf(m, part[i]);
    const float scale = block_scale(m), inv = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < kBlockSteps; ++i)
        if (row0 + kBlockStep * i < rows && col < cols)
            __stcs(reinterpret_cast<uint2*>(q + (row0 + kBlockStep * i) * cols + col), quantize8(v[i], inv));
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
}

// ---------------------------------------------------------------------------
// Combine: out[t] = sum_j weights[t,j] * rows[row_of[t,j]], f32 sums in the order of j, rounded once.
// Without weights it is the gradient of dispatch.  A warp takes U x 512 bytes of one token and keeps
// four rows' loads in flight.
// ---------------------------------------------------------------------------
template <typename T, int U, bool WEIGHTED>
__global__ void __launch_bounds__(kThreads) combine_kernel(MoveArgs a) {
    pdl_prologue();
    constexpr int N = Vec<T>::kN;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t t = unit / a.segs;
    if (t >= a.tokens) return;
    const int v0 = (int)(unit - t * a.segs) * 32 * U + lane;
    const uint4* rows = reinterpret_cast<const uint4*>(a.src);
    int my_row = -1;
    float my_w = 1.0f;
    if (lane < a.top_k) {
        my_row = __ldg(a.row_of + t * a.top_k + lane);
        if (WEIGHTED) my_w = __ldg(a.weights + t * a.top_k + lane);
    }
    if (my_row >= a.rows) my_row = -1;
    float acc[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[u][i] = 0.0f;
    constexpr int kGroup = 4;
    for (int j0 = 0; j0 < a.top_k; j0 += kGroup) {
        uint4 d[kGroup][U];
        int r[kGroup];
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            r[g] = j0 + g < a.top_k ? __shfl_sync(0xffffffffu, my_row, j0 + g) : -1;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r[g] >= 0 && v0 + 32 * u < a.vecs) d[g][u] = ld_stream(rows + (int64_t)r[g] * a.vecs + v0 + 32 * u);
        }
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            if (r[g] < 0) continue;
            const float w = WEIGHTED ? __shfl_sync(0xffffffffu, my_w, j0 + g) : 1.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[N];
                Vec<T>::unpack(d[g][u], f);
#pragma unroll
                for (int i = 0; i < N; ++i) acc[u][i] = WEIGHTED ? fmaf(w, f[i], acc[u][i]) : acc[u][i] + f[i];
            }
        }
    }
    uint4* out = reinterpret_cast<uint4*>(a.dst) + t * a.vecs;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (v0 + 32 * u < a.vecs) st_stream(out + v0 + 32 * u, Vec<T>::pack(acc[u]));
}

// ---------------------------------------------------------------------------
// Combine backward: d_rows[r] = weights[t,j] * grad[t] (zeros where no entry owns r) and
// d_weights[t,j] = <rows[r], grad[t]>.  A CTA takes one token: its gradient is read once and held in
// registers while the k rows stream by.  Partial dot products go lane -> warp (shuffles) -> CTA
// (shared memory, one slot for each warp and choice), always in the same order.
// ---------------------------------------------------------------------------
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) combine_bwd_kernel(MoveArgs a) {
    pdl_prologue();
    constexpr int N = Vec<T>::kN;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4* d_rows = reinterpret_cast<uint4*>(a.d_rows);
    const int64_t zero_blocks = (a.zero_units + kWarps - 1) / kWarps;
    if (blockIdx.x < zero_blocks) {
        const int64_t unit = (int64_t)blockIdx.x * kWarps + warp;
        if (unit < a.zero_units) {
            const int seg = (int)(unit % a.segs);
            zero_unowned(d_rows, a.entry_of, unit / a.segs * 32, a.rows, a.vecs, seg * 128, min(a.vecs, (seg + 1) * 128), lane);
        }
        return;
    }
    __shared__ float part[kMaxTopK][kWarps];
    const int64_t t = (int64_t)blockIdx.x - zero_blocks;
    const uint4* grad = reinterpret_cast<const uint4*>(a.grad) + t * a.vecs;
    const uint4* rows = reinterpret_cast<const uint4*>(a.src);
    int my_row = -1;
    float my_w = 0.0f;
    if (lane < a.top_k) {
        my_row = __ldg(a.row_of + t * a.top_k + lane);
        my_w = __ldg(a.weights + t * a.top_k + lane);
    }
    if (my_row >= a.rows) my_row = -1;
    for (int j = lane; j < a.top_k; j += 32) part[j][warp] = 0.0f;
    __syncwarp();
    for (int base = 0; base < a.vecs; base += kThreads * U) {
        const int v0 = base + threadIdx.x;
        uint4 graw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            graw[u] = v0 + kThreads * u < a.vecs ? ld_stream(grad + v0 + kThreads * u) : make_uint4(0, 0, 0, 0);
        float g[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) Vec<T>::unpack(graw[u], g[u]);
        for (int j = 0; j < a.top_k; ++j) {
            const int r = __shfl_sync(0xffffffffu, my_row, j);
            if (r < 0) continue;
            const float w = __shfl_sync(0xffffffffu, my_w, j);
            uint4 d[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (v0 + kThreads * u < a.vecs) d[u] = ld_stream(rows + (int64_t)r * a.vecs + v0 + kThreads * u);
            float dot = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (v0 + kThreads * u >= a.vecs) continue;
                float f[N], o[N];
                Vec<T>::unpack(d[u], f);
#pragma unroll
                for (int i = 0; i < N; ++i) { dot = fmaf(f[i], g[u][i], dot); o[i] = w * g[u][i]; }
                st_stream(d_rows + (int64_t)r * a.vecs + v0 + kThreads * u, Vec<T>::pack(o));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (lane == 0) part[j][warp] += dot;
        }
    }
    __syncthreads();
    if (threadIdx.x < a.top_k) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += part[threadIdx.x][w];
        a.d_weights[t * a.top_k + threadIdx.x] = s;
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Threads of a CTA: few entries and experts are sorted sooner by few warps, which meet at every barrier (graph
// replay: 16 entries over 8 experts 2.6 us, with 1024 threads 3.3; 128 over 128 3.2 and 3.4; but 512 over 128 3.85
// and 3.5, 256 over 256 4.3 and 3.9).
int route_threads(int64_t n, int64_t experts) {
    return n <= kRouteFewEntries && experts <= kRouteFewExperts ? kRouteFewThreads : kRouteThreads;
}
int route_ctas(int64_t n) {
    // One CTA ranks 32 entries a warp and step; a second CTA costs a cluster barrier, which is less than a second
    // step (2048 entries over 64 experts: 4.6 us on two CTAs, 5.3 on one; 1024 over 32: 4.4 and 4.0).
    int ctas = 1;
    while (ctas < kRouteMaxCtas && n > (int64_t)ctas * kRouteThreads) ctas *= 2;
    return ctas;
}
int64_t route_per_warp(int64_t n, int64_t ctas, int threads) { return ceil_div(ceil_div(n, ctas * (threads / 32)), 32) * 32; }
size_t route_smem(int64_t n, int64_t experts) {
    if (n > kRouteClusterEntries) return (size_t)(kRouteThreads / 32) * experts * sizeof(int);
    const int threads = route_threads(n, experts), warps = threads / 32;
    return ((size_t)(warps + 5) * experts + (experts & 1)) * sizeof(int) + (size_t)route_per_warp(n, route_ctas(n), threads) * warps * sizeof(int2);
}
constexpr int kRouteMaxSmem = (kRouteThreads / 32 + 5) * kMaxExperts * (int)sizeof(int) + kRouteThreads * kRouteRegSteps * (int)sizeof(int2);
static_assert(kRouteMaxSmem + 64 * (int)sizeof(int) <= 227 * 1024, "shared memory of the route kernel");

bool is_bf16(const Record& r) { return (r.flags & PB200_F_OUT_BF16) != 0; }

// Steps of a warp (each `step` wide) over a row of `width`: the most, up to `most`, that still leave a few warps
// for every SM sub-partition (short calls are bound by latency, long ones by bytes in flight) and at most an eighth
// of the row's last segment beyond its end (1000 rows of 2064 bf16 quantised: 3.1 us with two steps, 3.9 with four).
int pick_steps(int64_t rows, int64_t width, int64_t step, int most) {
    int u = most;
    while (u > 1 && (rows * ceil_div(width, step * u) < (int64_t)sm_count() * 16 || ceil_div(width, step * u) * step * u * 8 > width * 9)) u /= 2;
    return u;
}

// How a movement or row-quantising kernel walks its rows of `width` (16-byte vectors, or columns where it quantises):
// `steps` of a warp make a segment, `zero_units` clear 32 rows' segments each, `grid` CTAs in all.
struct Walk {
    int64_t width, segs, zero_units, grid;
};
Walk walk_of(const Record& r, int steps) {
    const int64_t T = r.dims[0], H = r.dims[3];
    const int64_t vecs = H * ((r.flags & PB200_F_OUT_BF16) ? 2 : 4) / 16;
    Walk w{};
    switch (r.kernel_id) {
    case PB200_K_FP8_QUANTIZE:
    case PB200_K_MOE_DISPATCH_FP8:
        w.width = r.kernel_id == PB200_K_FP8_QUANTIZE ? r.dims[1] : H;
        w.segs = ceil_div(w.width, 256 * steps);
        break;
    case PB200_K_MOE_COMBINE_BWD:                   // a CTA a token; its segments are those of the rows to clear
        w.width = vecs;
        w.segs = ceil_div(vecs, 128);
        break;
    default:
        w.width = vecs;
        w.segs = ceil_div(vecs, 32 * steps);
    }
    const bool clears = r.kernel_id == PB200_K_MOE_DISPATCH || r.kernel_id == PB200_K_MOE_DISPATCH_FP8 || r.kernel_id == PB200_K_MOE_COMBINE_BWD;
    w.zero_units = clears ? ceil_div(r.dims[2], 32) * w.segs : 0;
    w.grid = r.kernel_id == PB200_K_MOE_COMBINE_BWD ? ceil_div(w.zero_units, kWarps) + T : ceil_div(w.zero_units + T * w.segs, kWarps);
    return w;
}
// The steps of a handle, chosen when it is made.
int steps_of(const Record& r) {
    const int64_t width = walk_of(r, 1).width;
    switch (r.kernel_id) {
    case PB200_K_FP8_QUANTIZE:
    case PB200_K_MOE_DISPATCH_FP8: return pick_steps(r.dims[0], width, 256, 4);
    case PB200_K_MOE_DISPATCH:     return pick_steps(r.dims[0], width, 32, 4);
    case PB200_K_MOE_COMBINE_BWD:  return 4;
    default:                       return pick_steps(r.dims[0], width, 32, 2);
    }
}

template <typename... KArgs, typename... Args>
int enqueue(const char* what, void (*kernel)(KArgs...), const Record& r, cudaStream_t stream, char* err, Args... args) {
    cudaError_t e = launch_with_pdl(kernel, dim3(r.geom.grid[0]), dim3(r.geom.block[0]), 0, stream, args...);
    if (e != cudaSuccess) { set_err(err, "%s launch failed: %s", what, cudaGetErrorString(e)); return PB200_ERR_LAUNCH; }
    return PB200_OK;
}

template <typename IdT>
int launch_route(const Record& r, cudaStream_t stream, void** p, char* err) {
    RouteArgs a;
    a.ids = p[0];
    a.row_of = (int*)p[1];
    a.entry_of = (int*)p[2];
    a.offsets = (int*)p[3];
    const int64_t n = r.dims[0] * r.dims[1];
    a.n = (int)n;
    a.experts = (int)r.dims[2];
    a.block = (int)r.dims[3];
    a.rows = (int)r.dims[4];
    const bool wide = n > kRouteClusterEntries;
    const int ctas = (int)r.geom.grid[0], threads = (int)r.geom.block[0];
    a.per_warp = (int)route_per_warp(n, ctas, threads);
    const int form = threads == kRouteFewThreads ? 0 : 1;
    auto kernel = form == 0 ? route_kernel<IdT, kRouteFewThreads> : route_kernel<IdT, kRouteThreads>;
    const size_t smem = route_smem(n, a.experts);
    static std::atomic<uint64_t> attr_set[3];       // bit per device, for the kernels of this id type
    std::atomic<uint64_t>& done = attr_set[wide ? 2 : form];
    cudaError_t e = cudaSuccess;
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(done.load(std::memory_order_relaxed) & (1ull << (dev & 63)))) {
        // The limit belongs to the kernel, not to a launch: one for all sizes, since another thread may launch another size.
        e = wide ? cudaFuncSetAttribute(route_rank_kernel<IdT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRouteMaxSmem)
                 : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRouteMaxSmem);
        if (e == cudaSuccess) done.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
    if (e == cudaSuccess && wide) {
        int* counts = (int*)p[4];
        e = launch_with_pdl(route_rank_kernel<IdT>, dim3(ctas), dim3(threads), smem, stream, a, counts);
        if (e == cudaSuccess) e = launch_with_pdl(route_place_kernel<IdT>, dim3(ctas), dim3(threads), 0, stream, a, (const int*)counts);
    } else if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    if (e != cudaSuccess) { set_err(err, "moe_route launch failed: %s", cudaGetErrorString(e)); return PB200_ERR_LAUNCH; }
    return PB200_OK;
}

MoveArgs move_args(const Record& r, int64_t width, int elt_bytes) {
    MoveArgs a{};
    a.tokens = r.dims[0];
    a.top_k = (int)r.dims[1];
    a.rows = (int)r.dims[2];
    a.width = (int)width;
    a.vecs = (int)(width * elt_bytes / 16);
    a.scale_cols = (int)ceil_div(width, kScaleBlock);
    const Walk w = walk_of(r, r.steps);
    a.segs = (int)w.segs;
    a.zero_units = w.zero_units;
    return a;
}

template <typename T, bool ROUTED>
int launch_quantize_rows(const Record& r, MoveArgs a, cudaStream_t stream, char* err) {
    auto kernel = r.steps == 4 ? quantize_rows_kernel<T, 4, ROUTED> : r.steps == 2 ? quantize_rows_kernel<T, 2, ROUTED> : quantize_rows_kernel<T, 1, ROUTED>;
    return enqueue("fp8 quantisation", kernel, r, stream, err, a);
}

template <typename T, bool WEIGHTED>
int launch_combine(const Record& r, MoveArgs a, cudaStream_t stream, char* err) {
    return enqueue("moe_combine", r.steps == 1 ? combine_kernel<T, 1, WEIGHTED> : combine_kernel<T, 2, WEIGHTED>, r, stream, err, a);
}

}  // namespace

int plan_moe(Record& r, char* err) {
    auto bad = [&](const char* what) { set_err(err, "%s", what); return PB200_ERR_BAD_SHAPE; };
    pb200_geometry& g = r.geom;
    for (int i = 0; i < 3; ++i) g.grid[i] = g.block[i] = g.cluster[i] = 1;
    g.block[0] = kThreads;
    const int need = r.kernel_id == PB200_K_FP8_QUANTIZE ? 3 : r.kernel_id == PB200_K_MOE_ROUTE ? 5 : 4;
    if (r.n_dims != need) { set_err(err, "kernel %d needs %d dims, got %d", r.kernel_id, need, r.n_dims); return PB200_ERR_BAD_SHAPE; }
    for (int i = 0; i < need; ++i) {
        if (r.dims[i] < 1) return bad("all sizes must be positive");
        if (r.dims[i] > kMaxExtent) return bad("extent exceeds 2^31-65536");
    }
    if (r.kernel_id == PB200_K_FP8_QUANTIZE) {
        const int64_t M = r.dims[0], K = r.dims[1];
        if (K % 16 != 0) { set_err(err, "K=%lld must be divisible by 16", (long long)K); return PB200_ERR_BAD_SHAPE; }
        if (r.dims[2] != 1 && r.dims[2] != kScaleBlock) return bad("block_rows must be 1 or 128");
        const int64_t grid = r.dims[2] == 1 ? ceil_div(M * ceil_div(K, 256), kWarps) : ceil_div(M, kScaleBlock) * ceil_div(K, kScaleBlock);
        if (grid > 0x7fffffffLL) return bad("matrix is too large for one launch");
        if (r.dims[2] == 1) {
            r.steps = steps_of(r);
            g.grid[0] = (uint32_t)walk_of(r, r.steps).grid;
        } else {
            g.grid[0] = (uint32_t)grid;
            g.block[0] = kBlockThreads;
        }
        g.n_inputs = 1;
        g.n_outputs = 2;
        return PB200_OK;
    }
    const int64_t T = r.dims[0], k = r.dims[1];
    if (k > kMaxTopK) { set_err(err, "top_k=%lld exceeds %d", (long long)k, kMaxTopK); return PB200_ERR_BAD_SHAPE; }
    if (T * k > (1LL << 30)) return bad("tokens * top_k exceeds 2^30");
    if (r.kernel_id == PB200_K_MOE_ROUTE) {
        const int64_t E = r.dims[2], block = r.dims[3], rows = r.dims[4];
        if (E > kMaxExperts) { set_err(err, "E=%lld exceeds %d", (long long)E, kMaxExperts); return PB200_ERR_BAD_SHAPE; }
        if (block > kMaxBlock) { set_err(err, "block=%lld exceeds %d", (long long)block, kMaxBlock); return PB200_ERR_BAD_SHAPE; }
        if (rows % block != 0) { set_err(err, "rows=%lld must be divisible by block=%lld", (long long)rows, (long long)block); return PB200_ERR_BAD_SHAPE; }
        const int64_t n = T * k;
        if (n > kRouteClusterEntries) {
            g.grid[0] = (uint32_t)ceil_div(n, route_per_warp(n, sm_count(), kRouteThreads) * (kRouteThreads / 32));
            g.scratch_bytes = (uint64_t)E * g.grid[0] * sizeof(int);
        } else {
            g.cluster[0] = g.grid[0] = (uint32_t)route_ctas(n);
        }
        g.block[0] = (uint32_t)route_threads(n, E);
        g.smem_bytes = (uint32_t)route_smem(n, E);
        g.n_inputs = 1;
        g.n_outputs = 3;
        return PB200_OK;
    }
    const int64_t rows = r.dims[2], H = r.dims[3];
    const bool fp8 = r.kernel_id == PB200_K_MOE_DISPATCH_FP8;
    const int unit = fp8 ? 16 : is_bf16(r) ? 8 : 4;
    if (H % unit != 0) { set_err(err, "H=%lld must be divisible by %d", (long long)H, unit); return PB200_ERR_BAD_SHAPE; }
    // one warp for each 32 vectors at most, and the same again for rows to clear
    if (ceil_div(T + ceil_div(rows, 32), 1) * ceil_div(H, 128) > 0x7fffffffLL) return bad("tensor is too large for one launch");
    r.steps = steps_of(r);
    g.grid[0] = (uint32_t)walk_of(r, r.steps).grid;
    switch (r.kernel_id) {
        case PB200_K_MOE_DISPATCH:     g.n_inputs = 3; g.n_outputs = 1; break;
        case PB200_K_MOE_DISPATCH_FP8: g.n_inputs = 3; g.n_outputs = 2; break;
        case PB200_K_MOE_DISPATCH_BWD: g.n_inputs = 2; g.n_outputs = 1; break;
        case PB200_K_MOE_COMBINE:      g.n_inputs = 3; g.n_outputs = 1; break;
        default:                       g.n_inputs = 5; g.n_outputs = 2; break;
    }
    return PB200_OK;
}

int launch_moe(const Record& r, cudaStream_t stream, void** p, char* err) {
    const bool b16 = is_bf16(r), in_b16 = (r.flags & PB200_F_IN_BF16) != 0;
    switch (r.kernel_id) {
    case PB200_K_MOE_ROUTE:
        return (r.flags & PB200_F_IDS_S64) ? launch_route<int64_t>(r, stream, p, err) : launch_route<int32_t>(r, stream, p, err);
    case PB200_K_MOE_DISPATCH: {
        MoveArgs a = move_args(r, r.dims[3], b16 ? 2 : 4);
        a.src = p[0]; a.row_of = (const int*)p[1]; a.entry_of = (const int*)p[2]; a.dst = p[3];
        return enqueue("moe_dispatch", r.steps == 1 ? dispatch_kernel<1> : r.steps == 2 ? dispatch_kernel<2> : dispatch_kernel<4>, r, stream, err, a);
    }
    case PB200_K_MOE_DISPATCH_FP8: {
        MoveArgs a = move_args(r, r.dims[3], 1);
        a.src = p[0]; a.row_of = (const int*)p[1]; a.entry_of = (const int*)p[2]; a.dst = p[3]; a.dst_scale = (float*)p[4];
        return in_b16 ? launch_quantize_rows<__nv_bfloat16, true>(r, a, stream, err) : launch_quantize_rows<float, true>(r, a, stream, err);
    }
    case PB200_K_MOE_DISPATCH_BWD: {
        MoveArgs a = move_args(r, r.dims[3], b16 ? 2 : 4);
        a.row_of = (const int*)p[0]; a.src = p[1]; a.dst = p[2];
        return b16 ? launch_combine<__nv_bfloat16, false>(r, a, stream, err) : launch_combine<float, false>(r, a, stream, err);
    }
    case PB200_K_MOE_COMBINE: {
        MoveArgs a = move_args(r, r.dims[3], b16 ? 2 : 4);
        a.src = p[0]; a.weights = (const float*)p[1]; a.row_of = (const int*)p[2]; a.dst = p[3];
        return b16 ? launch_combine<__nv_bfloat16, true>(r, a, stream, err) : launch_combine<float, true>(r, a, stream, err);
    }
    case PB200_K_MOE_COMBINE_BWD: {
        MoveArgs a = move_args(r, r.dims[3], b16 ? 2 : 4);
        a.src = p[0]; a.weights = (const float*)p[1]; a.row_of = (const int*)p[2]; a.entry_of = (const int*)p[3]; a.grad = p[4];
        a.d_rows = p[5]; a.d_weights = (float*)p[6];
        return b16 ? enqueue("moe_combine_bwd", combine_bwd_kernel<__nv_bfloat16, 4>, r, stream, err, a)
                   : enqueue("moe_combine_bwd", combine_bwd_kernel<float, 4>, r, stream, err, a);
    }
    default: break;
    }
    // PB200_K_FP8_QUANTIZE
    const int64_t M = r.dims[0], K = r.dims[1];
    if (r.dims[2] == 1) {
        MoveArgs a{};
        a.tokens = M; a.width = (int)K; a.scale_cols = (int)ceil_div(K, kScaleBlock); a.segs = (int)walk_of(r, r.steps).segs;
        a.src = p[0]; a.dst = p[1]; a.dst_scale = (float*)p[2];
        return in_b16 ? launch_quantize_rows<__nv_bfloat16, false>(r, a, stream, err) : launch_quantize_rows<float, false>(r, a, stream, err);
    }
    const int sc = (int)ceil_div(K, kScaleBlock);
    if (in_b16)
        return enqueue("fp8 quantisation", quantize_blocks_kernel<__nv_bfloat16>, r, stream, err, (const __nv_bfloat16*)p[0],
                       (uint8_t*)p[1], (float*)p[2], M, (int)K, sc);
    return enqueue("fp8 quantisation", quantize_blocks_kernel<float>, r, stream, err, (const float*)p[0], (uint8_t*)p[1],
                   (float*)p[2], M, (int)K, sc);
}

}  // namespace pb200
