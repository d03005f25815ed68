// q4k_lora.cu -- q4k_lora_batch: low-rank adapters of many requests beside
// the shared projections of a step.
//
//   u[j][t]   = scale_a * sum_k A_a[t][k] x[j][k]        (shrink)
//   dst[j][n] = base[j][n] + sum_t B_a[n][t] u[j][t]     (expand), a = ids[j]
#include "q4k_device.cuh"
#include "q4k_internal.h"
#include "q4k_request.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

using namespace q4k;
namespace cg = cooperative_groups;

namespace {

struct LoraTask {
    const float *x, *base;
    float *dst;
    const void *A, *B;
    const int32_t *ranks;
    const float *scales;
    int64_t sx, sbase, sdst, sa_slot, sa_row, sb_slot, sb_row;
    int K, nrows, slots, rank;
    int u_off;  // first value of this task in a column's u (a multiple of 8)
};

// Columns of one adapter that are worked on together (many columns).
struct LoraTile {
    int slot, first, count;  // slot (-1: no adapter), first place in the sorted order, columns
};

struct LoraParams {
    LoraTask task[Q4K_MAX_TASKS];
    const int32_t *ids;
    int ntasks, ncols;
    // many columns only: workspace and splits
    int *status;  // the workspace's status word
    int *ntiles;
    LoraTile *tiles;
    int *order;   // columns sorted by adapter
    uint16_t *u;  // three bf16 pieces of u: 3 x ncols x u_cols, in sorted order
    int u_cols, splits, max_slots, rows_per_cta;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ int slot_of(const LoraTask &t, int id) { return id >= 0 && id < t.slots ? id : -1; }
__device__ __forceinline__ int rank_of(const LoraTask &t, int a) {
    if (t.ranks == nullptr) return t.rank;
    const int r = t.ranks[a];
    return r < 0 ? 0 : r > t.rank ? t.rank : r;
}

// ---- few columns: one cluster per adapter and group of columns -------------------
// The A and B of a column's adapter are the bytes of the call (1 MB at rank 64,
// 4096 x 4096, 16 bits), and a step's calls are too short for two launches. One
// launch: the cluster splits K over its CTAs (each reads its slice of every row
// of A once), the partial u meet over distributed shared memory, and each CTA
// expands its slice of the rows of B. Where there are more columns than
// clusters run at once, columns of one adapter share the reading: the cluster
// of every G-th column of an adapter takes the next G of them, the clusters of
// the others end at once.
// What bounds it is the chain of round trips to memory, so it is kept short:
// ids -> rank -> {scale, x, first A, first B, base} -> partial sums -> cluster
// barrier -> the other CTAs' parts -> rows. (Asking for A and B before the rank
// is known, as far as the slots have room, gained nothing and cost 1 us at K =
// 14336.) In a graph: one column through
// 4096 x 4096, rank 16, bf16 4.8 us (an empty launch takes about 2); 8 columns
// of 3 adapters, K = 14336, rank 32, fp32 8.7 us; 64 columns of 16 adapters,
// 14336 rows 25 us. The same sums on bf16 MMAs (below) measured slower here
// (one column 5.6, K = 14336 in fp32 11.8 us): cutting weights into pieces
// costs more than it saves where a weight serves one to four columns.
// 512 threads on an SM measured faster than two CTAs of 256 where a call has
// bytes to move (8 columns, K = 14336, fp32: 9.4 against 11.4 us), with 64
// registers for two CTAs of 512 it spills (9.5 -> 12.3 us).
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kClusterCols = 64;  // columns up to which this kernel runs (bits of a mask)
constexpr int kTile = 1024;       // values of x per column in shared memory at a time
constexpr int kBatch = 2;         // rows of A per warp and pass
constexpr int kAhead = 4;         // chunks of a row of B in flight per lane

// V values of T as they lie in memory; V * sizeof(T) is 16 (one load) or V is 1.
template <typename T, int V> struct alignas(V > 1 ? 16 : sizeof(T)) Chunk {
    T v[V];
};
template <typename T, int V> __device__ __forceinline__ Chunk<T, V> zero_chunk() {
    Chunk<T, V> c;
#pragma unroll
    for (int e = 0; e < V; ++e) c.v[e] = T(0.0f);
    return c;
}
// Values [0, n) of a row at p, n >= 1; the rest is zero and not read. The ends
// of rows go out of line: inlined at every load they made the code several
// times as long, and a short call waits for its instructions.
template <typename T, int V> __device__ __noinline__ Chunk<T, V> load_end(const T *p, int n) {
    Chunk<T, V> c = zero_chunk<T, V>();
#pragma unroll
    for (int e = 0; e < V - 1; ++e)
        if (e < n) c.v[e] = p[e];
    return c;
}
template <typename T, int V> __device__ __forceinline__ Chunk<T, V> load_chunk(const T *p, int n) {
    if constexpr (V > 1) {
        if (n < V) return load_end<T, V>(p, n);
        // (volatile: asked for where it stands, not where it is used)
        uint4 raw;
        asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "l"(p));
        return *reinterpret_cast<const Chunk<T, V> *>(&raw);
    } else {
        Chunk<T, V> c;
        c.v[0] = __ldg(p);
        return c;
    }
}

// Sums of M (a power of two, at most 32) values over the warp in M + log2(32 / M) - 1
// exchanges: each step halves the values a lane still holds. Lane l ends with
// the sum of value l / (32 / M).
template <int M> __device__ __forceinline__ float warp_sums(float (&v)[M], int lane) {
    int o = 16;
#pragma unroll
    for (int m = M; m > 1; m /= 2, o /= 2) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < m / 2; ++i) {
            const float mine = up ? v[i + m / 2] : v[i], other = up ? v[i] : v[i + m / 2];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
    }
    float s = v[0];
#pragma unroll
    for (; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// The columns of one group: the lowest G bits of `mask` (fewer where it has fewer).
template <typename T, int VA, int VB, int G, int NC>
__device__ __forceinline__ void lora_group(const LoraTask &t, int a, int r, uint64_t mask, float *xs, float *part,
                                           float *us, cg::cluster_group &cluster) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int me = static_cast<int>(cluster.block_rank());
    int col[G];  // -1: none
#pragma unroll
    for (int g = 0; g < G; ++g) {
        col[g] = __ffsll(static_cast<long long>(mask)) - 1;
        mask &= mask - 1;
    }
    const T *A = static_cast<const T *>(t.A) + a * t.sa_slot;
    const T *B = static_cast<const T *>(t.B) + a * t.sb_slot;
    const float scale = t.scales != nullptr ? t.scales[a] : 1.0f;

    // shrink: this CTA's slice [k0, k1) of K, a warp per kBatch rows, the next chunks asked for ahead
    const int kper = ((t.K + NC - 1) / NC + 7) / 8 * 8;
    const int k0 = min(t.K, me * kper), k1 = min(t.K, k0 + kper);
    for (int i = tid; i < r * G; i += kThreads) part[i] = 0.0f;
    const int passes = (r + kWarps * kBatch - 1) / (kWarps * kBatch);

    // expand: L lanes per row (one where the slice has rows for all threads)
    const int nper = (t.nrows + NC - 1) / NC;
    const int n0 = min(t.nrows, me * nper), n1 = min(t.nrows, n0 + nper);
    int L = 1;
    while (L < 32 && L * VB < r && 2 * L * nper <= kThreads) L *= 2;
    const int sub = tid & (L - 1), rows = kThreads / L;
    int n = n0 + tid / L;
    Chunk<T, VB> wb[kAhead];
    float base[G];
    auto ask = [&](int c0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = c0 + i * L * VB;
            // (a chunk that begins below r is read as far as the row has room; values behind r are not used)
            wb[i] = n < n1 && c < r ? load_chunk<T, VB>(B + n * t.sb_row + c, t.rank - c) : zero_chunk<T, VB>();
        }
    };
    auto ask_base = [&]() {
#pragma unroll
        for (int g = 0; g < G; ++g)
            base[g] = t.base != nullptr && n < n1 && col[g] >= 0 && sub == (g & (L - 1)) ? t.base[col[g] * t.sbase + n] : 0.0f;
    };

    for (int k = k0; k < k1; k += kTile) {
        const int kt = min(kTile, k1 - k);
        const int chunks = (kt + 32 * VA - 1) / (32 * VA);
        auto load = [&](Chunk<T, VA> (&w)[kBatch], int pass, int chunk) {
            const int c = (chunk * 32 + lane) * VA;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int q = pass * kWarps * kBatch + i * kWarps + warp;
                w[i] = q < r && c < kt ? load_chunk<T, VA>(A + q * t.sa_row + k + c, kt - c) : zero_chunk<T, VA>();
            }
        };
        Chunk<T, VA> w[kBatch];
        load(w, 0, 0);
        __syncthreads();  // the tile before this one is done with
        for (int i = tid; i < chunks * 32 * VA; i += kThreads)  // (zeros where a last chunk reads on)
#pragma unroll
            for (int g = 0; g < G; ++g) xs[g * kTile + i] = col[g] >= 0 && i < kt ? t.x[col[g] * t.sx + k + i] : 0.0f;
        if (k == k0) {
            ask(sub * VB);
            ask_base();
        }
        __syncthreads();
        float acc[kBatch * G] = {};
        for (int pass = 0, chunk = 0; pass < passes;) {
            const int np = chunk + 1 < chunks ? pass : pass + 1, nx = chunk + 1 < chunks ? chunk + 1 : 0;
            Chunk<T, VA> next[kBatch];
            if (np < passes) load(next, np, nx);
            const int c = (chunk * 32 + lane) * VA;
#pragma unroll
            for (int e = 0; e < VA; ++e)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        acc[i * G + g] = fmaf(to_f32(w[i].v[e]), xs[g * kTile + c + e], acc[i * G + g]);
            if (nx == 0) {
                const float s = warp_sums<kBatch * G>(acc, lane);
                constexpr int kLanes = 32 / (kBatch * G);
                const int v = lane / kLanes, q = pass * kWarps * kBatch + v / G * kWarps + warp;
                if (lane % kLanes == 0 && q < r) part[q * G + v % G] += s;
#pragma unroll
                for (int i = 0; i < kBatch * G; ++i) acc[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) w[i] = next[i];
            pass = np;
            chunk = nx;
        }
    }
    if (k0 >= k1) {  // (no slice of K here)
        ask(sub * VB);
        ask_base();
    }
    cluster.sync();
    for (int i = tid; i < (r + VB - 1) / VB * VB * G; i += kThreads) {  // (zeros behind the rank)
        float p[NC], s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) p[c] = i < r * G ? cluster.map_shared_rank(part, c)[i] : 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) s += p[c];
        us[i] = s * scale;
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // this CTA has read the others' parts
    __syncthreads();
    for (int nb = n0; nb < n1; nb += rows) {  // (uniform: lanes without a row take part in the exchanges)
        float acc[G] = {};
        for (int c0 = sub * VB;;) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int c = c0 + i * L * VB;
                if (c >= r) break;
                if (VB > 1 && c + VB > r)  // values behind the rank may be anything (u is zero there)
#pragma unroll
                    for (int e = 1; e < VB; ++e)
                        if (c + e >= r) wb[i].v[e] = T(0.0f);
#pragma unroll
                for (int e = 0; e < VB; ++e)
#pragma unroll
                    for (int g = 0; g < G; ++g) acc[g] = fmaf(to_f32(wb[i].v[e]), us[(c + e) * G + g], acc[g]);
            }
            c0 += kAhead * L * VB;
            if (c0 - sub * VB >= r) break;
            ask(c0);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            for (int o = L / 2; o > 0; o /= 2) acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], o);
            if (col[g] >= 0 && n < n1 && sub == (g & (L - 1))) t.dst[col[g] * t.sdst + n] = base[g] + acc[g];
        }
        n += rows;
        if (nb + rows < n1) {
            ask(sub * VB);
            ask_base();
        }
    }
    // no CTA leaves while another may still read its part
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int VA, int VB, int G, int NC>
__global__ void __launch_bounds__(kThreads) k_lora_cluster(const __grid_constant__ LoraParams P) {
    extern __shared__ __align__(16) float smem[];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait();
    const LoraTask &t = P.task[blockIdx.y];
    const int j = blockIdx.x / NC;
    const int tid = threadIdx.x, lane = tid & 31;
    // the columns that have this column's adapter, as a mask
    const int id0 = lane < P.ncols ? P.ids[lane] : -1, id1 = lane + 32 < P.ncols ? P.ids[lane + 32] : -1;
    const int a = slot_of(t, __shfl_sync(0xffffffffu, j < 32 ? id0 : id1, j & 31));
    const int r = a < 0 ? 0 : rank_of(t, a);
    if (r == 0) {  // nothing to add: the column's rows are base's
        const int me = static_cast<int>(cluster.block_rank());
        const int nper = (t.nrows + NC - 1) / NC;
        const int n0 = min(t.nrows, me * nper), n1 = min(t.nrows, n0 + nper);
        for (int n = n0 + tid; n < n1; n += kThreads)
            t.dst[j * t.sdst + n] = t.base != nullptr ? t.base[j * t.sbase + n] : 0.0f;
        return;  // (the whole cluster takes this way)
    }
    uint64_t mask = __ballot_sync(0xffffffffu, id0 == a) | static_cast<uint64_t>(__ballot_sync(0xffffffffu, id1 == a)) << 32;
    const uint64_t before = mask & ((uint64_t(1) << j) - 1);
    if (__popcll(before) % G != 0) return;  // another column's cluster does this one (all CTAs agree)
    mask &= ~before;
    float *xs = smem, *part = smem + G * kTile, *us = part + G * ((t.rank + 3) & ~3);  // (16-byte aligned)
    lora_group<T, VA, VB, G, NC>(t, a, r, mask, xs, part, us, cluster);
}

size_t cluster_smem(int g, int rank) { return (g * kTile + 2 * static_cast<size_t>(g) * (rank + 8)) * sizeof(float); }

template <typename T, int VA, int VB, int G, int NC>
cudaError_t launch_cluster_of(const LoraParams &p, int ntasks, int rank, cudaStream_t s) {
    auto *fn = k_lora_cluster<T, VA, VB, G, NC>;
    static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cluster_smem(G, Q4K_MAX_LORA_RANK)));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    return launch_request(fn, dim3(p.ncols * NC, ntasks), kThreads, cluster_smem(G, rank), dim3(NC), p, s);
}

template <typename T, int VA, int VB>
cudaError_t launch_cluster(const LoraParams &p, int ntasks, int rank, cudaStream_t s) {
    // One CTA fits on an SM; by the times of calls of one cluster more, 7 clusters of 16, 15 of 8 or 33 of 4 run at once.
    // As long as a cluster for every column and task fits, sharing an adapter's bytes (they are in L2) gains less than the
    // columns' arithmetic on one cluster costs; beyond that the clusters shrink, and then columns share. Which columns
    // have one adapter is not known here. Measured in a graph, us:
    // 8 and 9 columns: clusters of 16 against 8: 4096 x 4096 rank 16 bf16 8.5 / 5.3, 1024 rows rank 8 7.9 / 4.7, 14336 rows
    // rank 32 13.4 / 10.8; K = 14336 in fp32, 2.4 MB of weights each: 14.8 / 13.8 and 15.8 / 16.0, and 8.7 / 13.6 where
    // one of 8 columns has no adapter, so these keep 16.
    // 16 and 18 columns: clusters of 8 against 4: 9.7 / 7.2, rank 64 18.6 / 15.2, 14336 rows 20.2 / 17.0, 14336 in fp32 34.9 / 33.2.
    // 24 (8 columns of q, k, v, rank 64 fp16): clusters of 4 15.2 with one adapter, 16.3 with eight; of 8 in groups of 2
    // 10.7 and 18.2.
    // 36 (12 columns of q, k, v): clusters of 4 19.4 with one adapter, 23.6 with twelve; in groups of 2 16.6 and 25.5.
    // 48 columns of 16 adapters, 4096 rows: clusters of 8 in groups of 4 14.5, of 4 in groups of 2 10.9.
    // 56 (8 columns of 7 projections, rank 16, eight adapters): clusters of 4 in groups of 4 18.3, one by one 13.5; 64 columns
    // of 16 adapters at random, 14336 rows: in groups of 4 24.8, of 2 31.5.
    const int pieces = p.ncols * ntasks;
    int64_t bytes = 0;  // of weights per piece
    for (int i = 0; i < ntasks; ++i)
        bytes = std::max<int64_t>(bytes, (p.task[i].K + static_cast<int64_t>(p.task[i].nrows)) * p.task[i].rank * sizeof(T));
    return pieces <= 7 || (pieces <= 9 && bytes >= 2000000) ? launch_cluster_of<T, VA, VB, 1, 16>(p, ntasks, rank, s)
           : pieces <= 15 ? launch_cluster_of<T, VA, VB, 1, 8>(p, ntasks, rank, s)
           : pieces <= 37 ? launch_cluster_of<T, VA, VB, 1, 4>(p, ntasks, rank, s)
           : pieces <= 48 ? launch_cluster_of<T, VA, VB, 2, 4>(p, ntasks, rank, s)
                          : launch_cluster_of<T, VA, VB, 4, 4>(p, ntasks, rank, s);
}

// ---- many columns: grouped products on the tensor cores ----------------------------
// Three launches: the columns are sorted by adapter into tiles of up to 64
// columns of one adapter; shrink computes u for a tile, K split over CTAs;
// expand adds the parts of u, and streams base -> dst. What has to move is x,
// base and dst once (A and B are small and stay in L2), so both products only
// have to keep up with memory. fp32 FMAs would not (4.3 GFLOP at rank 64,
// 4096 columns, 4096 x 4096: 60 us against 31 us of traffic); tf32 and plain
// bf16 would lose digits. So every fp32 value is cut into three bf16 pieces
// that add up to it exactly (8 bits each), an fp16 weight into two, and the
// products of pieces down to 2^-16 of the largest are summed on bf16 MMAs
// (3 for bf16 weights, 5 for fp16, 6 for fp32); what is left out is below an
// fp32 rounding: two products of a second and a third piece, 2^-8 x 2^-17
// each, of either sign. The MMAs' own sums are cut off, not rounded, so they
// are taken over into fp32 sums: by the shrink after at most 12 of them, by the
// expand after a chunk of 64 ranks (at most 24, the small products first).
// Terms of one sign come out 1.5 x 2^-24 off at any rank and type (3 for fp32
// weights while pieces were cut off; the rounding costs no time); one sum over
// the whole rank was 15 off at rank 128 and 88 at 512 (bf16 weights), and 1 to
// 3 % faster there.
constexpr int kTileCols = 64;  // columns per tile
constexpr int kRanks = 64;     // ranks per shrink CTA
constexpr int kStageK = 64;    // values of K per stage of A in shared memory
constexpr int kRing = 3;

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two fp32 values as sums of bf16 pieces, a's in the lower half: each piece rounded to nearest, so that what is left
// of it is at most 2^-8 of the value before (three pieces hold all 24 bits, two an fp16's 11) and of either sign.
template <int N> __device__ __forceinline__ void pieces(float a, float b, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const __nv_bfloat162 near = __floats2bfloat162_rn(a, b);
        p[i] = *reinterpret_cast<const uint32_t *>(&near);
        a -= __uint_as_float(p[i] << 16);
        b -= __uint_as_float(p[i] & 0xffff0000u);
    }
}
// An infinity cut into pieces becomes inf, NaN, NaN, and times another's zero piece NaN; values of kTop on round to
// an infinite piece. So what the MMAs give as infinite or NaN is summed anew from the values themselves: it comes out as the fp32 sum, as with few columns.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
template <typename T> __device__ __noinline__ float plain_dot(const T *a, const float *x, int K) {
    float s = 0.0f;
    for (int k = 0; k < K && s == s; k += 8)  // (NaN stays: columns of NaN end at once)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) s = fmaf(to_f32(a[k + e]), x[k + e], s);
    return s;
}
template <typename T> __device__ __noinline__ float plain_sum(const T *b, const uint16_t *u, int64_t piece, int r) {
    auto value = [&](int64_t i) { return __uint_as_float(static_cast<uint32_t>(u[i]) << 16); };
    float s = 0.0f;
#pragma unroll 1
    for (int k = 0; k < r && s == s; ++k) s = fmaf(to_f32(b[k]), value(k) + (value(piece + k) + value(2 * piece + k)), s);
    return s;
}
// Pieces that add up to any value: the first holds what is not finite, and of values of kTop on the upper half.
constexpr float kTop = 0x1.ffp127f;
__device__ __noinline__ uint3 whole_pieces(float a, float b) {
    auto rest = [](float v) { return fabsf(v) < kTop ? v : finite(v) ? v - __uint_as_float(__float_as_uint(v) & 0xffff0000u) : 0.0f; };
    auto first = [](float v) { return v != v ? 0x7fff0000u : __float_as_uint(v) & 0xffff0000u; };
    uint32_t p[3];
    pieces(rest(a), rest(b), p);
    const bool ta = !(fabsf(a) < kTop), tb = !(fabsf(b) < kTop);
    if (ta) p[2] = (p[2] & 0xffff0000u) | (p[1] & 0xffffu), p[1] = (p[1] & 0xffff0000u) | (p[0] & 0xffffu), p[0] = (p[0] & 0xffff0000u) | first(a) >> 16;
    if (tb) p[2] = (p[2] & 0xffffu) | (p[1] & 0xffff0000u), p[1] = (p[1] & 0xffffu) | (p[0] & 0xffff0000u), p[0] = (p[0] & 0xffffu) | first(b);
    return make_uint3(p[0], p[1], p[2]);
}
template <typename T> struct Weight;  // bf16 pieces of a weight
template <> struct Weight<__nv_bfloat16> { static constexpr int kPieces = 1; };
template <> struct Weight<__half> { static constexpr int kPieces = 2; };
template <> struct Weight<float> { static constexpr int kPieces = 3; };

// Eight consecutive weights as MMA operands: q[piece][i] holds weights 2i, 2i + 1.
template <typename T> struct Eight {
    T v[8];
};
template <typename T> __device__ __forceinline__ void weights(const Eight<T> &w, uint32_t (&q)[Weight<T>::kPieces][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Weight<T>::kPieces == 1) {
            q[0][i] = *reinterpret_cast<const uint32_t *>(&w.v[2 * i]);
        } else {
            uint32_t p[Weight<T>::kPieces];
            pieces(to_f32(w.v[2 * i]), to_f32(w.v[2 * i + 1]), p);
#pragma unroll
            for (int k = 0; k < Weight<T>::kPieces; ++k) q[k][i] = p[k];
        }
    }
}
template <typename T> __device__ __forceinline__ Eight<T> load_eight_smem(const T *p) {
    Eight<T> w;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        reinterpret_cast<uint4 *>(&w)[i] = reinterpret_cast<const uint4 *>(p)[i];
    return w;
}
// Values [0, n) at p (n may be 0 or less), the others zero. V: p is 16-byte aligned.
template <typename T, bool V> __device__ __forceinline__ Eight<T> load_eight(const T *p, int n) {
    Eight<T> w;
    if (V && n >= 8) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            reinterpret_cast<uint4 *>(&w)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w.v[e] = e < n ? p[e] : T(0.0f);
    }
    return w;
}

// acc = the products of 16 rows of fp32 pieces with 4 x 8 rows of weights over
// 32 values each: weight(b) gives lane (g, q) its eight weights of row g of the
// b-th eight. The small products come first; the four sums are independent, so
// their MMAs follow one another without waiting.
template <typename T, typename F>
__device__ __forceinline__ void products(float (&acc)[4][4], const uint32_t (&a)[2][3][4], F weight) {
    constexpr int N = Weight<T>::kPieces;
    uint32_t wq[4][N][4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        weights(weight(b), wq[b]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[b][e] = 0.0f;
    }
#pragma unroll
    for (int order = 2; order >= 0; --order)
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k <= order)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int b = 0; b < 4; ++b) mma_bf16(acc[b], a[m][order - k], wq[b][k][2 * m], wq[b][k][2 * m + 1]);
}

// Sorts the columns by adapter (bins: the slots, then "none") and lists the tiles.
__global__ void __launch_bounds__(1024) k_lora_plan(const __grid_constant__ LoraParams P) {
    __shared__ int bin[Q4K_MAX_LORA_SLOTS + 1], at[Q4K_MAX_LORA_SLOTS + 1], warps[2][32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, bins = P.max_slots + 1;
    auto bin_of = [&](int j) {
        const int id = P.ids[j];
        return id >= 0 && id < P.max_slots ? id : P.max_slots;
    };
    // one addition per warp and bin
    auto add = [&](int *counts, int j) {
        const bool live = j < P.ncols;
        const int b = live ? bin_of(j) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, b);
        const int lead = __ffs(same) - 1;
        int first = 0;
        if (live && lane == lead) first = atomicAdd(&counts[b], __popc(same));
        return __shfl_sync(0xffffffffu, first, lead) + __popc(same & ((1u << lane) - 1));
    };
    for (int i = tid; i < bins; i += 1024) bin[i] = 0;
    __syncthreads();
    for (int j0 = tid - lane; j0 < P.ncols; j0 += 1024) add(bin, j0 + lane);
    __syncthreads();
    // exclusive sums over the bins: columns and tiles before each (bins <= 1025: thread 0 takes the last one too)
    int c[2] = {0, 0}, upto[2];
    const int mine = tid < bins ? bin[tid] : 0;
    c[0] = mine;
    c[1] = (mine + kTileCols - 1) / kTileCols;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        upto[k] = c[k];
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto[k], o);
            if (lane >= o) upto[k] += v;
        }
        if (lane == 31) warps[k][tid / 32] = upto[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (int w = 0; w < tid / 32; ++w) upto[k] += warps[k][w];
    auto list = [&](int b, int cols, int first, int tile) {
        at[b] = first;
        for (int i = 0; i < cols; i += kTileCols)
            P.tiles[tile++] = {b < P.max_slots ? b : -1, first + i, min(kTileCols, cols - i)};
        if (b == bins - 1) {
            *P.ntiles = tile;
            *P.status = Q4K_OK;
        }
    };
    if (tid < bins) list(tid, mine, upto[0] - c[0], upto[1] - c[1]);
    if (tid == 1023 && bins == 1025) list(1024, bin[1024], upto[0], upto[1]);
    __syncthreads();
    for (int j0 = tid - lane; j0 < P.ncols; j0 += 1024) {
        const int p = add(at, j0 + lane);
        if (j0 + lane < P.ncols) P.order[p] = j0 + lane;
    }
}

__device__ __forceinline__ void cp_async16(void *dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void cp_async4(void *dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src),
                 "r"(bytes)
                 : "memory");
}

// Stage of the shrink's ring: kStageK values of kTileCols columns of x, and of
// kRanks rows of A as kStageK / 32 slabs of 32. Pitches let the eight rows and
// four eights of a fragment load meet different banks.
constexpr int kXPitch = kStageK + 4;
constexpr int kStageValues = kRanks * kStageK;
template <typename T> constexpr size_t kShrinkStage = kTileCols * kXPitch * 4 + kStageValues * sizeof(T);
constexpr int kMaxSplits = 16;  // CTAs that share a tile's K: a cluster

// u of a tile's columns for kRanks ranks. The cluster splits K; in a CTA four
// pairs of warps take 16 columns each, a warp one half of every stage. x and A come through a ring; lane q of a row
// takes eights of consecutive values of both, so the MMAs sum over the same
// pairs whatever their order. The CTAs' sums meet over distributed shared
// memory, and u leaves as the pieces that the expand's MMAs take.
template <typename T, bool VX, bool VA>
__global__ void __launch_bounds__(256, 2) k_lora_shrink(const __grid_constant__ LoraParams P) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ const float *xcol[kTileCols];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait();
    if (static_cast<int>(blockIdx.x) >= *P.ntiles) return;  // (the whole cluster, here and below)
    const LoraTile tile = P.tiles[blockIdx.x];
    int z = blockIdx.z, ti = 0;
    while (z >= (P.task[ti].rank + kRanks - 1) / kRanks) z -= (P.task[ti++].rank + kRanks - 1) / kRanks;
    const LoraTask &t = P.task[ti];
    const int a = slot_of(t, tile.slot), r = a < 0 ? 0 : rank_of(t, a), r0 = z * kRanks;
    if (r0 >= r) return;
    const int nr = min(kRanks, r - r0), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q = lane & 3, m0 = (warp & 3) * 16, half = warp >> 2;
    if (tid < tile.count) xcol[tid] = t.x + P.order[tile.first + tid] * t.sx;
    __syncthreads();
    // this CTA's share of K: whole stages
    const int stages = (t.K + kStageK - 1) / kStageK, per = (stages + P.splits - 1) / P.splits;
    const int s0 = min(stages, static_cast<int>(blockIdx.y) * per), s1 = min(stages, s0 + per);
    const bool busy = m0 < tile.count;
    const T *A = static_cast<const T *>(t.A) + a * t.sa_slot + r0 * t.sa_row;
    auto fill = [&](int s) {
        float *xs = reinterpret_cast<float *>(smem_raw + (s % kRing) * kShrinkStage<T>);
        T *as = reinterpret_cast<T *>(xs + kTileCols * kXPitch);
        if (s < s1) {
            const int k0 = s * kStageK;
            if constexpr (VX) {
                const int k = tid % 16 * 4, left = min(4, t.K - k0 - k);
                for (int row = tid / 16; row < tile.count; row += 16)
                    cp_async16(xs + row * kXPitch + k, left > 0 ? xcol[row] + k0 + k : xcol[row], left > 0 ? left * 4 : 0);
            } else {
                const int k = tid % kStageK;
                const bool some = k0 + k < t.K;
                for (int row = tid / kStageK; row < tile.count; row += 256 / kStageK)
                    cp_async4(xs + row * kXPitch + k, some ? xcol[row] + k0 + k : xcol[row], some ? 4 : 0);
            }
            if constexpr (VA) {
                constexpr int E = 16 / sizeof(T), C = kStageK / E;  // values per copy, copies per row
                const int k = tid % C * E, left = min(E, t.K - k0 - k);
                for (int row = tid / C; row < kRanks; row += 256 / C) {
                    const bool some = left > 0 && row < nr;
                    cp_async16(as + ((k / 32) * kRanks + row) * 32 + k % 32, some ? A + row * t.sa_row + k0 + k : A,
                               some ? left * static_cast<int>(sizeof(T)) : 0);
                }
            } else {
                const int k = tid % kStageK;
                T v[kRanks * kStageK / 256];  // (all asked for before the first is stored)
#pragma unroll
                for (int i = 0; i < kRanks * kStageK / 256; ++i) {
                    const int row = tid / kStageK + i * (256 / kStageK);
                    v[i] = row < nr && k0 + k < t.K ? A[row * t.sa_row + k0 + k] : T(0.0f);
                }
#pragma unroll
                for (int i = 0; i < kRanks * kStageK / 256; ++i)
                    as[((k / 32) * kRanks + tid / kStageK + i * (256 / kStageK)) * 32 + k % 32] = v[i];
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float sum[8][4] = {};
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fill(s0 + i);
    for (int s = s0; s < s1; ++s) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        __syncthreads();  // stage s has come, and stage s - 1 may be written again
        fill(s + kRing - 1);
        if (!busy) continue;
        const float *xs = reinterpret_cast<const float *>(smem_raw + (s % kRing) * kShrinkStage<T>);
        const T *as = reinterpret_cast<const T *>(xs + kTileCols * kXPitch);
        uint32_t xa[2][3][4];  // [MMA][piece][operand registers]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // (rows behind the tile's columns hold anything: an MMA keeps rows apart)
            const Eight<float> x = load_eight_smem(xs + (m0 + g + 8 * h) * kXPitch + half * 32 + 8 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t p[3];
                pieces(x.v[2 * i], x.v[2 * i + 1], p);
#pragma unroll
                for (int k = 0; k < 3; ++k) xa[i / 2][k][(i % 2) * 2 + h] = p[k];
            }
        }
#pragma unroll
        for (int n = 0; n < 8; n += 4) {
            if (n * 8 >= nr) break;
            float acc[4][4];
            products<T>(acc, xa, [&](int b) { return load_eight_smem(as + (half * kRanks + (n + b) * 8 + g) * 32 + 8 * q); });
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[n + b][e] += acc[b][e];
        }
    }
    // the halves' sums, [half][column][rank], over the ring
    constexpr int kPitch = kRanks + 4;
    float *part = reinterpret_cast<float *>(smem_raw);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (busy)
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<float2 *>(part + (half * kTileCols + m0 + g + 8 * h) * kPitch + n * 8 + 2 * q) =
                    make_float2(sum[n][2 * h], sum[n][2 * h + 1]);
    cluster.sync();
    const float scale = t.scales != nullptr ? t.scales[a] : 1.0f;
    const int pairs = (nr + 7) / 8 * 4;  // (whole eights: zeros behind the rank)
    for (int i = blockIdx.y * 256 + tid; i < tile.count * (kRanks / 2); i += P.splits * 256) {
        const int col = i / (kRanks / 2), k = i % (kRanks / 2);
        if (k >= pairs) continue;
        float2 v = make_float2(0.0f, 0.0f);
        for (int c = 0; c < P.splits; ++c) {
            const float *from = cluster.map_shared_rank(part, c) + col * kPitch + 2 * k;
            const float2 w0 = *reinterpret_cast<const float2 *>(from);
            const float2 w1 = *reinterpret_cast<const float2 *>(from + kTileCols * kPitch);
            v.x += w0.x + w1.x;
            v.y += w0.y + w1.y;
        }
        const bool one = 2 * k < nr, two = 2 * k + 1 < nr;
        float2 w = make_float2(one ? v.x * scale : 0.0f, two ? v.y * scale : 0.0f);
        uint32_t p[3];
        if (fabsf(w.x) < kTop && fabsf(w.y) < kTop) {
            pieces(w.x, w.y, p);
        } else {
            if (one && !finite(v.x)) w.x = plain_dot(A + 2 * k * t.sa_row, xcol[col], t.K) * scale;
            if (two && !finite(v.y)) w.y = plain_dot(A + (2 * k + 1) * t.sa_row, xcol[col], t.K) * scale;
            const uint3 q3 = whole_pieces(w.x, w.y);
            p[0] = q3.x, p[1] = q3.y, p[2] = q3.z;
        }
#pragma unroll
        for (int e = 0; e < 3; ++e)
            *reinterpret_cast<uint32_t *>(P.u + (static_cast<int64_t>(e) * P.ncols + tile.first + col) * P.u_cols + t.u_off + r0 +
                                          2 * k) = p[e];
    }
    cluster.sync();  // no CTA leaves while another may still read its part
}

// ---- expand: 5th-generation tensor cores ------------------------------------------
// dst of a tile's columns for a range of rows, in tiles of 128 rows: D (128 rows
// x 64 columns, fp32 in tensor memory) = pieces of B (128 x 64 ranks, shared
// memory) x pieces of u (64 columns x 64 ranks). One thread issues the MMAs;
// afterwards a lane of tensor memory is a row, so a warp reads base and writes
// dst for 32 consecutive rows of a column at a time, whatever their alignment.
// Operands lie K-major in rows of 128 bytes, 16-byte units exchanged within a
// row by its index modulo 8 (the 128-byte swizzle).
constexpr int kRows = 128;                     // rows of a tile
constexpr int kChunkK = 64;                    // ranks of a chunk: one swizzled row of bf16
constexpr int kUBytes = kTileCols * 128;       // one piece of u's chunk
constexpr int kBBytes = kRows * 128;           // one piece of B's chunk
constexpr int kTmemCols = 64;                  // D; as many again for sums over several chunks
template <typename T> constexpr size_t kExpandSmem = 3 * kUBytes + Weight<T>::kPieces * kBBytes + 1024;  // (+ alignment)

__device__ __forceinline__ uint32_t swizzled(int row, int unit) { return row * 128 + ((unit ^ (row & 7)) << 4); }
// Shared-memory operand descriptor: K-major, 128-byte swizzle, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fff) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
           uint64_t(2) << 61;
}
// fp32 += bf16 x bf16, both operands K-major, M = 128, N = 64.
constexpr uint32_t kMmaShape = 1u << 4 | 1u << 7 | 1u << 10 | (kTileCols / 8) << 17 | (kRows / 16) << 24;
__device__ __forceinline__ void mma_tmem(uint32_t d, uint64_t a, uint64_t b, bool add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b),
        "r"(kMmaShape), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// 16 columns of this warp's 32 lanes.
__device__ __forceinline__ void load_tmem(uint32_t (&v)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr)
        : "memory");
}
// Sums kept beside D, eight columns of this warp's 32 lanes at a time.
__device__ __forceinline__ void load_tmem8(float (&v)[8], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void store_tmem8(uint32_t addr, const float (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
        "tcgen05.wait::st.sync.aligned;" ::"r"(addr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
        : "memory");
}
// Waits for a phase of the barrier, at most two seconds.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t until = globaltimer_ns() + 2000000000ull;
    while (!mbar_try_wait(bar, parity))
        if (globaltimer_ns() > until) return false;
    return true;
}

// Four CTAs per SM overlap one another's chain (operands -> MMAs -> base -> dst):
// 4096 columns took 73.1 us with three, 70.2 with four, 75.7 with five (whole call).
template <typename T, bool VB>
__global__ void __launch_bounds__(256, 4) k_lora_expand(const __grid_constant__ LoraParams P) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ struct {
        const float *base;
        float *dst;
    } col[kTileCols];
    __shared__ __align__(8) uint64_t done;  // the MMAs of a chunk
    __shared__ uint32_t tmem;
    pdl_launch_dependents();
    pdl_wait();
    if (static_cast<int>(blockIdx.x) >= *P.ntiles) return;
    const LoraTile tile = P.tiles[blockIdx.x];
    const LoraTask &t = P.task[blockIdx.z];
    const int n0 = blockIdx.y * P.rows_per_cta, n1 = min(t.nrows, n0 + P.rows_per_cta);
    if (n0 >= n1) return;
    const int a = slot_of(t, tile.slot), r = a < 0 ? 0 : rank_of(t, a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (r == 0) {  // nothing to add
        for (int i = warp; i < tile.count; i += 8) {
            const int64_t j = P.order[tile.first + i];
            for (int n = n0 + lane; n < n1; n += 32) t.dst[j * t.sdst + n] = t.base != nullptr ? t.base[j * t.sbase + n] : 0.0f;
        }
        return;
    }
    constexpr int N = Weight<T>::kPieces;
    uint8_t *us = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bs = us + 3 * kUBytes;
    if (tid < tile.count) {
        const int64_t j = P.order[tile.first + tid];
        col[tid] = {t.base != nullptr ? t.base + j * t.sbase : nullptr, t.dst + j * t.sdst};
    }
    __syncwarp();
    const int tmem_cols = r > kChunkK ? 2 * kTmemCols : kTmemCols;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem)), "r"(tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        if (lane == 0) {
            mbar_init(smem_addr(&done), 1);
            mbar_fence_init();
        }
    }
    const T *B = static_cast<const T *>(t.B) + a * t.sb_slot;
    const int chunks = (r + kChunkK - 1) / kChunkK, tiles = (n1 - n0 + kRows - 1) / kRows;
    // chunk c of u (columns behind the tile's: zeros) and of the rows of tile i of B; zeros behind the rank and the rows
    auto fill_u = [&](int c) {
        for (int i = tid; i < 3 * kTileCols * 8; i += 256) {
            const int unit = i & 7, row = (i >> 3) & (kTileCols - 1), piece = i / (8 * kTileCols), k = c * kChunkK + unit * 8;
            const bool some = row < tile.count && k < r;
            const uint16_t *u = some ? P.u + (static_cast<int64_t>(piece) * P.ncols + tile.first + row) * P.u_cols + t.u_off + k : P.u;
            cp_async16(us + piece * kUBytes + swizzled(row, unit), u, some ? 16 : 0);
        }
    };
    auto fill_b = [&](int i, int c) {
        const int row0 = n0 + i * kRows;
#pragma unroll
        for (int e = 0; e < kRows * 8 / 256; ++e) {
            const int unit = tid & 7, row = (tid >> 3) + e * 32, k = c * kChunkK + unit * 8;
            const int left = row0 + row < n1 ? r - k : 0;
            const T *from = B + (row0 + row) * t.sb_row + k;
            if constexpr (VB && N == 1) {
                cp_async16(bs + swizzled(row, unit), left > 0 ? from : B, left > 0 ? min(left, 8) * 2 : 0);
            } else {
                uint32_t q[N][4];
                weights(load_eight<T, VB>(from, left), q);
#pragma unroll
                for (int p = 0; p < N; ++p)
                    *reinterpret_cast<uint4 *>(bs + p * kBBytes + swizzled(row, unit)) = make_uint4(q[p][0], q[p][1], q[p][2], q[p][3]);
            }
        }
    };
    fill_u(0);
    fill_b(0, 0);
    bool bad = false;
    uint32_t parity = 0;
    for (int s = 0, i = 0, c = 0; i < tiles; ++s) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        // the operands have come, and (at first) the allocation; the tile before has been read out of tensor memory
        if (__syncthreads_or(bad)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem;
        if (tid == 0) {
            bool add = false;
#pragma unroll
            for (int order = 2; order >= 0; --order)  // small products first
#pragma unroll
                for (int p = 0; p < N; ++p)
                    if (p <= order)
#pragma unroll
                        for (int k = 0; k < kChunkK / 16; ++k) {
                            mma_tmem(d, operand(smem_addr(bs) + p * kBBytes) + 2 * k,
                                     operand(smem_addr(us) + (order - p) * kUBytes) + 2 * k, add);
                            add = true;
                        }
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(&done))
                         : "memory");
        }
        const bool last = c + 1 == chunks, first = c == 0;
        const int n = n0 + i * kRows + (warp & 3) * 32 + lane, c0 = warp / 4 * 32;
        float y[16];
        auto ask = [&](int from) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float *b = from + e < tile.count ? col[from + e].base : nullptr;
                y[e] = b != nullptr && n < n1 ? b[n] : 0.0f;
            }
        };
        if (last) ask(c0);
        bad = __any_sync(0xffffffffu, !wait_bounded(smem_addr(&done), parity));  // (a warp leaves as one)
        parity ^= 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        c = last ? 0 : c + 1;
        i += last;
        if (i < tiles && !bad) {  // (the MMAs are through with the operands)
            if (chunks > 1) fill_u(c);
            fill_b(i, c);
        }
        if (bad) continue;
        uint32_t mine = d + ((warp & 3) * 32 << 16) + c0;
        if (chunks > 1) {  // the chunk's sums are taken over into the kept ones
            __syncwarp();
#pragma unroll 1
            for (int k = 0; k < 32; k += 8) {
                float v[8], kept[8];
                load_tmem8(v, mine + k);
                if (!first) {
                    load_tmem8(kept, mine + kTmemCols + k);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += kept[e];
                }
                store_tmem8(mine + kTmemCols + k, v);
            }
            if (!last) continue;
            mine += kTmemCols;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t v[16];
            __syncwarp();
            load_tmem(v, mine + 16 * h);
            float probe = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) probe = fmaf(__uint_as_float(v[e]), 0.0f, probe);
            if (probe == 0.0f) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + 16 * h + e < tile.count && n < n1) col[c0 + 16 * h + e].dst[n] = y[e] + __uint_as_float(v[e]);
                if (h == 0) ask(c0 + 16);
                continue;
            }
            uint32_t anew = 0u;  // columns whose sum is not finite
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool ok = finite(__uint_as_float(v[e]));
                if (!ok) anew |= 1u << e;
                if (ok && c0 + 16 * h + e < tile.count && n < n1) col[c0 + 16 * h + e].dst[n] = y[e] + __uint_as_float(v[e]);
            }
            for (; anew != 0u; anew &= anew - 1) {
                const int e = c0 + 16 * h + __ffs(anew) - 1;
                if (e >= tile.count || n >= n1) continue;
                const uint16_t *u = P.u + static_cast<int64_t>(tile.first + e) * P.u_cols + t.u_off;
                const float s = plain_sum(B + n * t.sb_row, u, static_cast<int64_t>(P.ncols) * P.u_cols, r);
                col[e].dst[n] = (col[e].base != nullptr ? col[e].base[n] : 0.0f) + s;
            }
            if (h == 0) ask(c0 + 16);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bad) st_relaxed_gpu(P.status, Q4K_ETIMEOUT);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols));
    }
}

template <typename T> constexpr size_t kShrinkSmem = kRing * kShrinkStage<T>;
// Tiles there can be: whole ones, and one begun per bin.
int most_tiles(int ncols, int max_slots) { return ncols / kTileCols + (ncols < max_slots + 1 ? ncols : max_slots + 1); }

template <typename T>
cudaError_t launch_grouped(const LoraParams &p, bool vx, bool va, bool vb, cudaStream_t s) {
    auto *shrink = vx ? va ? k_lora_shrink<T, true, true> : k_lora_shrink<T, true, false>
                      : va ? k_lora_shrink<T, false, true> : k_lora_shrink<T, false, false>;
    auto *expand = vb ? k_lora_expand<T, true> : k_lora_expand<T, false>;
    static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        const int ss = static_cast<int>(kShrinkSmem<T>), es = static_cast<int>(kExpandSmem<T>);
        for (auto *f : {k_lora_shrink<T, true, true>, k_lora_shrink<T, true, false>, k_lora_shrink<T, false, true>,
                        k_lora_shrink<T, false, false>}) {
            if ((e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, ss)) != cudaSuccess) return e;
            if ((e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        }
        for (auto *f : {k_lora_expand<T, true>, k_lora_expand<T, false>})
            if ((e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, es)) != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    const unsigned tiles = static_cast<unsigned>(most_tiles(p.ncols, p.max_slots));
    if ((e = launch_request(k_lora_plan, dim3(1), 1024, 0, dim3(0), p, s)) != cudaSuccess) return e;
    unsigned chunks = 0, rows = 0;
    for (int i = 0; i < p.ntasks; ++i) {
        chunks += (p.task[i].rank + kRanks - 1) / kRanks;
        rows = std::max(rows, static_cast<unsigned>(p.task[i].nrows));
    }
    if (chunks > 0) {
        e = launch_request(shrink, dim3(tiles, p.splits, chunks), 256, kShrinkSmem<T>, dim3(1, p.splits), p, s);
        if (e != cudaSuccess) return e;
    }
    return launch_request(expand, dim3(tiles, (rows + p.rows_per_cta - 1) / p.rows_per_cta, p.ntasks), 256, kExpandSmem<T>,
                          dim3(0), p, s);
}

// Whether every run of 8 values of every row is 16-byte aligned.
bool rows_aligned(const void *p, int64_t slot, int64_t row, int esz) {
    return aligned_to(p, 16) && slot * esz % 16 == 0 && row * esz % 16 == 0;
}

template <typename T> cudaError_t launch_lora(const LoraParams &p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    bool va = true, vb = true, vx = true;
    int rank = 0;
    for (int i = 0; i < p.ntasks; ++i) {
        const LoraTask &t = p.task[i];
        va = va && rows_aligned(t.A, t.sa_slot, t.sa_row, sizeof(T));
        vb = vb && rows_aligned(t.B, t.sb_slot, t.sb_row, sizeof(T));
        vx = vx && rows_aligned(t.x, 0, t.sx, 4);
        rank = std::max(rank, t.rank);
    }
    if (p.ncols > kClusterCols) return launch_grouped<T>(p, vx, va, vb, s);
    const int n = p.ntasks;
    return va ? vb ? launch_cluster<T, V, V>(p, n, rank, s) : launch_cluster<T, V, 1>(p, n, rank, s)
              : vb ? launch_cluster<T, 1, V>(p, n, rank, s) : launch_cluster<T, 1, 1>(p, n, rank, s);
}

int type_bytes(int type) { return type == Q4K_TYPE_F32 ? 4 : type == Q4K_TYPE_F16 || type == Q4K_TYPE_BF16 ? 2 : 0; }

// fp32 columns of n values, `stride` values apart.
Runs columns(const float *p, int64_t n, int64_t stride, int ncols) { return {p, n * 4, stride * 4, ncols}; }

int check_task(const q4k_lora_task &t, int i, int ncols) {
    if (!extent_ok(t.K) || !extent_ok(t.nrows))
        return request_fail(Q4K_EINVAL, "task %d: K=%lld, nrows=%lld", i, (long long)t.K, (long long)t.nrows);
    if (t.slots < 0 || t.slots > Q4K_MAX_LORA_SLOTS)
        return request_fail(Q4K_EINVAL, "task %d: slots=%d outside 0..%d", i, t.slots, Q4K_MAX_LORA_SLOTS);
    if (t.rank < 0 || t.rank > Q4K_MAX_LORA_RANK)
        return request_fail(Q4K_EINVAL, "task %d: rank=%d outside 0..%d", i, t.rank, Q4K_MAX_LORA_RANK);
    const int esz = type_bytes(t.type);
    if (esz == 0) return request_fail(Q4K_EINVAL, "task %d: type=%d is not F32, F16 or BF16", i, t.type);
    if (ncols == 0 || t.nrows == 0) return Q4K_OK;
    if (t.dst == nullptr) return request_fail(Q4K_EINVAL, "task %d: null dst", i);
    if (!aligned_to(t.dst, 4) || !aligned_to(t.base, 4) || !aligned_to(t.x, 4) || !aligned_to(t.ranks, 4) ||
        !aligned_to(t.scales, 4))
        return request_fail(Q4K_EINVAL, "task %d: an fp32 or int32 pointer is not 4-byte aligned", i);
    if (!aligned_to(t.A, esz) || !aligned_to(t.B, esz))
        return request_fail(Q4K_EINVAL, "task %d: A or B is not aligned to its %d-byte type", i, esz);
    if (!stride_ok(t.stride_col_dst, ncols > 1 ? t.nrows : 0))
        return request_fail(Q4K_EINVAL, "task %d: stride_col_dst=%lld < nrows", i, (long long)t.stride_col_dst);
    if (t.base != nullptr) {
        if (!in_stride_ok(t.stride_col_base, ncols > 1 ? t.nrows : 0))
            return request_fail(Q4K_EINVAL, "task %d: stride_col_base=%lld < nrows", i, (long long)t.stride_col_base);
        const bool same = t.base == t.dst && (ncols == 1 || t.stride_col_base == t.stride_col_dst);
        if (!same && runs_overlap(columns(t.base, t.nrows, t.stride_col_base, ncols),
                                  columns(t.dst, t.nrows, t.stride_col_dst, ncols)))
            return request_fail(Q4K_EINVAL, "task %d: base overlaps dst without being dst", i);
    }
    if (t.K == 0 || t.slots == 0 || t.rank == 0) return Q4K_OK;  // dst = base: nothing else is read
    if (t.x == nullptr || t.A == nullptr || t.B == nullptr)
        return request_fail(Q4K_EINVAL, "task %d: null x, A or B", i);
    if (!in_stride_ok(t.stride_col_x, ncols > 1 ? t.K : 0))
        return request_fail(Q4K_EINVAL, "task %d: stride_col_x=%lld < K", i, (long long)t.stride_col_x);
    if (!stride_ok(t.stride_a_row, t.rank > 1 ? t.K : 0) ||
        !stride_ok(t.stride_a_slot, 0))
        return request_fail(Q4K_EINVAL, "task %d: strides of A (slot %lld, row %lld) too small for %d x %lld", i,
                            (long long)t.stride_a_slot, (long long)t.stride_a_row, t.rank, (long long)t.K);
    if (!stride_ok(t.stride_b_row, t.nrows > 1 ? t.rank : 0) ||
        !stride_ok(t.stride_b_slot, 0))
        return request_fail(Q4K_EINVAL, "task %d: strides of B (slot %lld, row %lld) too small for %lld x %d", i,
                            (long long)t.stride_b_slot, (long long)t.stride_b_row, (long long)t.nrows, t.rank);
    return Q4K_OK;
}

int check_tasks(const q4k_lora_task *tasks, int ntasks, int ncols) {
    if (ntasks < 0 || ntasks > Q4K_MAX_TASKS)
        return request_fail(Q4K_EINVAL, "ntasks=%d outside 0..%d", ntasks, Q4K_MAX_TASKS);
    if (!extent_ok(ncols)) return request_fail(Q4K_EINVAL, "ncols=%d < 0", ncols);
    if (ntasks > 0 && tasks == nullptr) return request_fail(Q4K_EINVAL, "null tasks");
    for (int i = 0; i < ntasks; ++i) {
        const int st = check_task(tasks[i], i, ncols);
        if (st != Q4K_OK) return st;
        if (tasks[i].type != tasks[0].type)
            return request_fail(Q4K_EINVAL, "task %d: type=%d differs from task 0's %d", i, tasks[i].type, tasks[0].type);
    }
    if (ncols == 0) return Q4K_OK;
    // the tasks run side by side: nothing one of them writes may be read or written by another
    for (int i = 0; i < ntasks; ++i) {
        if (tasks[i].nrows == 0) continue;
        const Runs w = columns(tasks[i].dst, tasks[i].nrows, tasks[i].stride_col_dst, ncols);
        for (int k = 0; k < ntasks; ++k) {
            const q4k_lora_task &r = tasks[k];
            if (r.x != nullptr && runs_overlap(w, columns(r.x, r.K, r.stride_col_x, ncols)))
                return request_fail(Q4K_EINVAL, "task %d: dst overlaps task %d's x", i, k);
            if (k == i || r.nrows == 0) continue;
            if (runs_overlap(w, columns(r.dst, r.nrows, r.stride_col_dst, ncols)))
                return request_fail(Q4K_EINVAL, "task %d: dst overlaps task %d's dst", i, k);
            if (r.base != nullptr && runs_overlap(w, columns(r.base, r.nrows, r.stride_col_base, ncols)))
                return request_fail(Q4K_EINVAL, "task %d: dst overlaps task %d's base", i, k);
        }
    }
    return Q4K_OK;
}

// Workspace of the many-column path: status word; behind the control words, which stay as they are (another call
// on the same workspace may rely on them): number of tiles; tiles; order; u.
struct LoraLayout {
    size_t ntiles = 0, tiles = 0, order = 0, u = 0, total = 0;
    int max_slots = 0, u_cols = 0, splits = 1;
};

LoraLayout lora_layout(const q4k_lora_task *tasks, int ntasks, int ncols) {
    LoraLayout L;
    if (ncols <= kClusterCols) return L;
    int64_t K = 0;
    for (int i = 0; i < ntasks; ++i) {
        if (tasks[i].nrows == 0) continue;
        L.max_slots = std::max(L.max_slots, tasks[i].slots);
        L.u_cols += (tasks[i].rank + 7) / 8 * 8;
        K = std::max(K, tasks[i].K);
    }
    // K is split until there are up to 256 CTAs (two fit on an SM: 4096 columns took 98.7 us at 256, 105.6 at 512, 108.5
    // at 150), but not below four stages
    const int64_t tiles = (ncols + kTileCols - 1) / kTileCols;
    L.splits = static_cast<int>(std::max<int64_t>(1, std::min({int64_t(kMaxSplits), 256 / tiles, K / (4 * kStageK)})));
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    L.ntiles = kControlBytes;
    L.tiles = L.ntiles + 256;
    L.order = L.tiles + up(static_cast<size_t>(most_tiles(ncols, L.max_slots)) * sizeof(LoraTile));
    L.u = L.order + up(static_cast<size_t>(ncols) * 4);
    L.total = L.u + up(static_cast<size_t>(3) * ncols * L.u_cols * 2);
    return L;
}

}  // namespace

extern "C" {

size_t q4k_lora_workspace_bytes(const q4k_lora_task *tasks, int ntasks, int ncols) {
    if (check_tasks(tasks, ntasks, ncols) != Q4K_OK) return 0;
    return lora_layout(tasks, ntasks, ncols).total;
}

int q4k_lora_batch(const q4k_lora_task *tasks, int ntasks, int ncols, const int32_t *ids, void *workspace,
                   size_t workspace_bytes, q4k_stream_t stream) {
    const int st = check_tasks(tasks, ntasks, ncols);
    if (st != Q4K_OK) return st;
    if (ncols == 0 || ntasks == 0) return Q4K_OK;
    if (ids == nullptr || !aligned_to(ids, 4)) return request_fail(Q4K_EINVAL, "ids null or not 4-byte aligned");
    const LoraLayout L = lora_layout(tasks, ntasks, ncols);
    const size_t need = L.total;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 256)))
        return request_fail(Q4K_EWORKSPACE, "workspace %p of %zu bytes; need %zu bytes, 256-byte aligned", workspace,
                            workspace_bytes, need);
    LoraParams p = {};
    int n = 0;
    for (int i = 0; i < ntasks; ++i) {
        const q4k_lora_task &t = tasks[i];
        if (t.nrows == 0) continue;
        const bool none = t.K == 0;
        LoraTask &d = p.task[n++];
        d = {t.x, t.base, t.dst, t.A, t.B, t.ranks, t.scales, t.stride_col_x, t.stride_col_base, t.stride_col_dst,
             t.stride_a_slot, t.stride_a_row, t.stride_b_slot, t.stride_b_row, static_cast<int>(t.K),
             static_cast<int>(t.nrows), none || t.rank == 0 ? 0 : t.slots, t.rank, p.u_cols};
        p.u_cols += (t.rank + 7) / 8 * 8;
    }
    if (n == 0) return Q4K_OK;
    p.ids = ids;
    p.ncols = ncols;
    p.ntasks = n;
    if (ncols > kClusterCols) {
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        p.status = reinterpret_cast<int *>(ws);
        p.ntiles = reinterpret_cast<int *>(ws + L.ntiles);
        p.tiles = reinterpret_cast<LoraTile *>(ws + L.tiles);
        p.order = reinterpret_cast<int *>(ws + L.order);
        p.u = reinterpret_cast<uint16_t *>(ws + L.u);
        p.splits = L.splits;
        p.max_slots = L.max_slots;
        // rows per expand CTA: few enough for several CTAs per SM
        int64_t rows = 0;
        for (int i = 0; i < n; ++i) rows += p.task[i].nrows;
        p.rows_per_cta = 512;
        const int64_t tiles = (ncols + kTileCols - 1) / kTileCols;
        while (p.rows_per_cta > kRows && tiles * (rows / p.rows_per_cta) < 592) p.rows_per_cta /= 2;
        while (rows / p.rows_per_cta >= 65535) p.rows_per_cta *= 2;  // (a grid's second dimension)
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = tasks[0].type == Q4K_TYPE_F32   ? launch_lora<float>(p, s)
                          : tasks[0].type == Q4K_TYPE_F16 ? launch_lora<__half>(p, s)
                                                          : launch_lora<__nv_bfloat16>(p, s);
    if (e != cudaSuccess) return request_cuda_fail(e, "lora launch");
    return Q4K_OK;
}

}  // extern "C"
