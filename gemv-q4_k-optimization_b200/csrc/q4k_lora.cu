// q4k_lora.cu -- q4k_lora_batch: low-rank adapters of many requests beside
// the shared projections of a step.
//
//   u[j][t]   = scale_a * sum_k A_a[t][k] x[j][k]        (shrink)
//   dst[j][n] = base[j][n] + sum_t B_a[n][t] u[j][t]     (expand), a = ids[j]
#include "q4k_request.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

using namespace q4k;

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

template <typename T>
cudaError_t launch_lora(const LoraParams &p, int ntasks, cudaStream_t s) {
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
