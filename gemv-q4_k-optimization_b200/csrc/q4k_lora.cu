// q4k_lora.cu -- q4k_lora_batch: low-rank adapters of many requests beside
// the shared projections of a step.
//
//   u[j][t]   = scale_a * sum_k A_a[t][k] x[j][k]        (shrink)
//   dst[j][n] = base[j][n] + sum_t B_a[n][t] u[j][t]     (expand), a = ids[j]
#include "q4k_request.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
    int u_off;  // first value of this task in a column's u
};

struct LoraParams {
    LoraTask task[Q4K_MAX_TASKS];
    const int32_t *ids;
    float *u;       // ncols x u_cols
    int u_cols;
    int ncols;
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

// One warp per (column, t): blockIdx.x = column, blockIdx.y = task, 8 warps over t.
template <typename T>
__global__ void __launch_bounds__(256) k_lora_shrink(const __grid_constant__ LoraParams P) {
    const LoraTask &t = P.task[blockIdx.y];
    const int64_t j = blockIdx.x;
    const int a = slot_of(t, P.ids[j]);
    if (a < 0) return;
    const int r = rank_of(t, a);
    const float scale = t.scales != nullptr ? t.scales[a] : 1.0f;
    const int lane = threadIdx.x & 31;
    const float *x = t.x + j * t.sx;
    for (int q = threadIdx.x >> 5; q < r; q += 8) {
        const T *row = static_cast<const T *>(t.A) + a * t.sa_slot + q * t.sa_row;
        float s = 0.0f;
        for (int k = lane; k < t.K; k += 32) s = fmaf(to_f32(row[k]), x[k], s);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) P.u[j * P.u_cols + t.u_off + q] = s * scale;
    }
}

// One thread per output: blockIdx.x = column, blockIdx.y = task, threads over rows.
template <typename T>
__global__ void __launch_bounds__(256) k_lora_expand(const __grid_constant__ LoraParams P) {
    const LoraTask &t = P.task[blockIdx.y];
    const int64_t j = blockIdx.x;
    const int a = slot_of(t, P.ids[j]);
    const int r = a < 0 ? 0 : rank_of(t, a);
    const float *u = P.u + j * P.u_cols + t.u_off;
    for (int n = blockIdx.z * 256 + threadIdx.x; n < t.nrows; n += gridDim.z * 256) {
        float s = 0.0f;
        if (r > 0) {
            const T *row = static_cast<const T *>(t.B) + a * t.sb_slot + n * t.sb_row;
            for (int q = 0; q < r; ++q) s = fmaf(to_f32(row[q]), u[q], s);
        }
        const float b = t.base != nullptr ? t.base[j * t.sbase + n] : 0.0f;
        t.dst[j * t.sdst + n] = b + s;
    }
}

// ---- few columns: one cluster per adapter and group of columns -------------------
// The A and B of a column's adapter are the bytes of the call (1 MB at rank 64,
// 4096 x 4096, 16 bits), and a step's calls are too short for two launches. One
// launch: the cluster splits K over its CTAs (each reads its slice of every row
// of A once), the partial u meet over distributed shared memory, and each CTA
// expands its slice of the rows of B. Columns that share an adapter share the
// reading: the cluster of every kGroup-th column of an adapter takes the next
// kGroup of them, the clusters of the others end at once.
// What bounds it is the chain of round trips to memory, so it is kept short:
// ids -> {ranks, scales, x, first A, first B, base} -> partial sums -> cluster
// barrier -> the other CTAs' parts -> rows.
#ifndef LORA_T
#define LORA_T 512
#define LORA_MB 1
#endif
constexpr int kThreads = LORA_T;
constexpr int kWarps = kThreads / 32;
constexpr int kClusterCols = 64;  // columns up to which this kernel runs (bits of a mask)
#ifndef LORA_G
#define LORA_G 8
#endif
constexpr int kGroup = LORA_G;         // columns of one adapter per cluster
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
// Values [0, n) of a row at p, n >= 1; the rest is zero and not read.
template <typename T, int V> __device__ __forceinline__ Chunk<T, V> load_chunk(const T *p, int n) {
    if constexpr (V > 1) {
        if (n >= V) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(p));
            return *reinterpret_cast<const Chunk<T, V> *>(&raw);
        }
        Chunk<T, V> c = zero_chunk<T, V>();
#pragma unroll
        for (int e = 0; e < V - 1; ++e)
            if (e < n) c.v[e] = p[e];
        return c;
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
            wb[i] = n < n1 && c < r ? load_chunk<T, VB>(B + n * t.sb_row + c, r - c) : zero_chunk<T, VB>();
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
    for (int i = tid; i < r * G; i += kThreads) {
        float p[NC], s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) p[c] = cluster.map_shared_rank(part, c)[i];
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
#pragma unroll
                for (int e = 0; e < VB; ++e)
                    if (c + e < r)
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

template <typename T, int VA, int VB, int NC>
__global__ void __launch_bounds__(kThreads, LORA_MB) k_lora_cluster(const __grid_constant__ LoraParams P) {
    extern __shared__ __align__(16) float smem[];
    cg::cluster_group cluster = cg::this_cluster();
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
    if (__popcll(before) % kGroup != 0) return;  // another column's cluster does this one (all CTAs agree)
    mask &= ~before;
    float *xs = smem, *part = smem + kGroup * kTile, *us = part + kGroup * t.rank;
    const int count = __popcll(mask);
    if (count == 1)
        lora_group<T, VA, VB, 1, NC>(t, a, r, mask, xs, part, us, cluster);
    else if (count <= 4)
        lora_group<T, VA, VB, 4, NC>(t, a, r, mask, xs, part, us, cluster);
    else
        lora_group<T, VA, VB, kGroup, NC>(t, a, r, mask, xs, part, us, cluster);
}

size_t cluster_smem(int rank) { return (kGroup * kTile + 2 * kGroup * rank) * sizeof(float); }

template <typename T, int VA, int VB, int NC>
cudaError_t launch_cluster_of(const LoraParams &p, int ntasks, int rank, cudaStream_t s) {
    auto *fn = k_lora_cluster<T, VA, VB, NC>;
    static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, cluster_smem(Q4K_MAX_LORA_RANK));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.ncols * NC, ntasks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = cluster_smem(rank);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = NC;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, p);
}

template <typename T, int VA, int VB>
cudaError_t launch_cluster(const LoraParams &p, int ntasks, int rank, cudaStream_t s) {
#ifdef LORA_NC
    return launch_cluster_of<T, VA, VB, LORA_NC>(p, ntasks, rank, s);
#else
    return p.ncols * ntasks <= 18 ? launch_cluster_of<T, VA, VB, 16>(p, ntasks, rank, s)
                                  : launch_cluster_of<T, VA, VB, 8>(p, ntasks, rank, s);
#endif
}

// Whether chunks of V values of every row are 16-byte aligned.
bool rows_aligned(const void *p, int64_t slot, int64_t row, int esz) {
    return aligned_to(p, 16) && slot * esz % 16 == 0 && row * esz % 16 == 0;
}

template <typename T>
cudaError_t launch_lora(const LoraParams &p, int ntasks, cudaStream_t s) {
    if (p.ncols <= kClusterCols) {
        constexpr int V = 16 / sizeof(T);
        bool va = true, vb = true;
        int rank = 0;
        for (int i = 0; i < ntasks; ++i) {
            const LoraTask &t = p.task[i];
            va = va && rows_aligned(t.A, t.sa_slot, t.sa_row, sizeof(T));
            vb = vb && rows_aligned(t.B, t.sb_slot, t.sb_row, sizeof(T));
            rank = t.rank > rank ? t.rank : rank;
        }
        return va ? vb ? launch_cluster<T, V, V>(p, ntasks, rank, s) : launch_cluster<T, V, 1>(p, ntasks, rank, s)
                  : vb ? launch_cluster<T, 1, V>(p, ntasks, rank, s) : launch_cluster<T, 1, 1>(p, ntasks, rank, s);
    }
    k_lora_shrink<T><<<dim3(p.ncols, ntasks), 256, 0, s>>>(p);
    k_lora_expand<T><<<dim3(p.ncols, ntasks, 8), 256, 0, s>>>(p);
    return cudaGetLastError();
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

size_t workspace_need(const q4k_lora_task *tasks, int ntasks, int ncols) {
    if (ncols <= kClusterCols) return 0;
    size_t u = 0;
    for (int i = 0; i < ntasks; ++i)
        if (tasks[i].nrows > 0) u += static_cast<size_t>(tasks[i].rank);
    return u * static_cast<size_t>(ncols) * sizeof(float);
}

}  // namespace

extern "C" {

size_t q4k_lora_workspace_bytes(const q4k_lora_task *tasks, int ntasks, int ncols) {
    if (check_tasks(tasks, ntasks, ncols) != Q4K_OK) return 0;
    return workspace_need(tasks, ntasks, ncols);
}

int q4k_lora_batch(const q4k_lora_task *tasks, int ntasks, int ncols, const int32_t *ids, void *workspace,
                   size_t workspace_bytes, q4k_stream_t stream) {
    const int st = check_tasks(tasks, ntasks, ncols);
    if (st != Q4K_OK) return st;
    if (ncols == 0 || ntasks == 0) return Q4K_OK;
    if (ids == nullptr || !aligned_to(ids, 4)) return request_fail(Q4K_EINVAL, "ids null or not 4-byte aligned");
    const size_t need = workspace_need(tasks, ntasks, ncols);
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
        p.u_cols += t.rank;
    }
    if (n == 0) return Q4K_OK;
    p.ids = ids;
    p.u = static_cast<float *>(workspace);
    p.ncols = ncols;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = tasks[0].type == Q4K_TYPE_F32   ? launch_lora<float>(p, n, s)
                          : tasks[0].type == Q4K_TYPE_F16 ? launch_lora<__half>(p, n, s)
                                                          : launch_lora<__nv_bfloat16>(p, n, s);
    if (e != cudaSuccess) return request_cuda_fail(e, "lora launch");
    return Q4K_OK;
}

}  // extern "C"
