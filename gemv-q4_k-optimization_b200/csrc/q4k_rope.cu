// q4k_rope.cu -- q4k_rope_multi: rotary positions with several axes on the
// query and key outputs of a step.
//
// Pair (a, b) of a head turns by phi = pos[axis][j] * inv_freq[i]:
//   (x_a, x_b) -> scale * (x_a cos - x_b sin, x_b cos + x_a sin).
// The angle is formed in fp64 as a number of half turns and reduced there
// (a far position times an inverse frequency holds more digits than fp32
// keeps). Its sine and cosine are fp32: those of the angle's fp32 part, turned
// by the remainder (at most 2^-25 half turns, so its first power is enough).
#include "q4k_device.cuh"
#include "q4k_request.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

using namespace q4k;

namespace {

struct RopeTensor {
    const float *x;
    void *dst;
    int64_t sx_col, sx_head, sd_col, sd_head;
    int heads;
};

struct RopeParams {
    RopeTensor t[Q4K_MAX_ROPE_TENSORS];
    const int32_t *pos;
    const double *inv_freq;
    int64_t sp_axis;
    int ntensors, head_dim, n_rot, n_axes, order, layout, sect_sum;
    int sect[Q4K_MAX_ROPE_AXES];
    float scale;
    int heads, lanes, heads_per_block;
};

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ int axis_of(const RopeParams &P, int i) {
    if (P.order == Q4K_ROPE_INTERLEAVED) {
        const int a = i % P.n_axes;
        return i / P.n_axes < P.sect[a] ? a : 0;
    }
    int r = i % P.sect_sum, a = 0;
    while (r >= P.sect[a]) r -= P.sect[a++];
    return a;
}

// Cosine and sine of pair i of column j, times the scale.
__device__ __forceinline__ float2 turn_of(const RopeParams &P, int i, int64_t j) {
    const double turns = static_cast<double>(P.pos[axis_of(P, i) * P.sp_axis + j]) * P.inv_freq[i] *
                         0.31830988618379067154;  // 1/pi: half turns
    const double r = turns - 2.0 * rint(0.5 * turns);
    const float near = static_cast<float>(r);
    const float left = static_cast<float>((r - static_cast<double>(near)) * 3.14159265358979323846);
    float s, c;
    sincospif(near, &s, &c);
    return make_float2(fmaf(-s, left, c) * P.scale, fmaf(c, left, s) * P.scale);
}

constexpr int kThreads = 256;

// Any sizes and strides: one block per column, one pair (or value behind the
// pairs) at a time. Bound by its 4-byte accesses and one division per pair: 8192
// columns of 40 heads of 126 take 92 us (0.55 of the measured copy rate), 8
// columns 4.3 us.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_rope(const __grid_constant__ RopeParams P) {
    __shared__ float2 cs[Q4K_MAX_ROPE_DIM / 2];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t j = blockIdx.x;
    const int half = P.n_rot / 2;
    for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = turn_of(P, i, j);
    __syncthreads();
    for (int k = 0; k < P.ntensors; ++k) {
        const RopeTensor &t = P.t[k];
        const float *x = t.x + j * t.sx_col;
        T *d = static_cast<T *>(t.dst) + j * t.sd_col;
        const int per = P.head_dim - half;  // pairs, then the values behind them
        for (int w = threadIdx.x; w < t.heads * per; w += kThreads) {
            const int h = w / per, i = w - h * per;
            const float *xh = x + h * t.sx_head;
            T *dh = d + h * t.sd_head;
            if (i < half) {
                const int a = P.layout == Q4K_ROPE_HALF ? i : 2 * i;
                const int b = P.layout == Q4K_ROPE_HALF ? i + half : 2 * i + 1;
                const float xa = xh[a], xb = xh[b];
                dh[a] = from_f32<T>(fmaf(xa, cs[i].x, -(xb * cs[i].y)));
                dh[b] = from_f32<T>(fmaf(xb, cs[i].x, xa * cs[i].y));
            } else {
                dh[half + i] = from_f32<T>(xh[half + i]);
            }
        }
    }
}

template <typename T> __device__ __forceinline__ void store4(T *d, const float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(d) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        T t[4] = {from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(t);
    }
}

// Heads of whole groups of four pairs (and of eight values behind them), all
// 16-byte aligned. What has to move is x and dst once; the angles cost one
// fp64 product and one sine per pair and column. A block takes a column and a
// share of its heads (of all tensors, one after the other); a thread keeps one
// group of four pairs, so its cosines and sines stay in registers, and walks
// over the heads. Its first values are asked for before the angles are formed.
// 8192 columns of 40 heads of 128: 55.4 us, 6.06 TB/s, 0.92 of the measured
// copy rate (value by value, k_rope took 95 us); 8 columns: 2.0 us.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kThreads) k_rope_vec(const __grid_constant__ RopeParams P) {
    __shared__ float2 cs[Q4K_MAX_ROPE_DIM / 2];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t j = blockIdx.x;
    const int half = P.n_rot / 2, groups = half / 4 + (P.head_dim - P.n_rot) / 8;
    const int g = threadIdx.x & (P.lanes - 1), step = kThreads / P.lanes;  // lanes: groups, up to a power of two
    const bool live = g < groups, pairs = g * 4 < half;
    // the group's two runs of four values
    const int lo = !pairs ? P.n_rot + (g - half / 4) * 8 : HALF ? g * 4 : g * 8;
    const int hi = pairs && HALF ? lo + half : lo + 4;
    int h = blockIdx.y * P.heads_per_block + threadIdx.x / P.lanes;
    const int h1 = min(P.heads, static_cast<int>(blockIdx.y + 1) * P.heads_per_block);
    auto tensor_of = [&](int &head) {
        int k = 0;
        while (head >= P.t[k].heads) head -= P.t[k++].heads;
        return k;
    };
    float4 a, b;
    auto load = [&](int head) {
        const RopeTensor &t = P.t[tensor_of(head)];
        const float *x = t.x + j * t.sx_col + head * t.sx_head;
        a = *reinterpret_cast<const float4 *>(x + lo);
        b = *reinterpret_cast<const float4 *>(x + hi);
    };
    if (live && h < h1) load(h);
    for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = turn_of(P, i, j);
    __syncthreads();
    if (!live) return;
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = pairs ? cs[g * 4 + i].x : 1.0f;
        s[i] = pairs ? cs[g * 4 + i].y : 0.0f;
    }
    for (; h < h1; h += step) {
        // values (a, b) of the four pairs: two runs, or neighbours
        float xa[4] = {a.x, HALF ? a.y : a.z, HALF ? a.z : b.x, HALF ? a.w : b.z};
        float xb[4] = {HALF ? b.x : a.y, HALF ? b.y : a.w, HALF ? b.z : b.y, b.w};
        float ya[4], yb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ya[i] = pairs ? fmaf(xa[i], c[i], -(xb[i] * s[i])) : xa[i];
            yb[i] = pairs ? fmaf(xb[i], c[i], xa[i] * s[i]) : xb[i];
        }
        int head = h;
        const RopeTensor &t = P.t[tensor_of(head)];
        T *d = static_cast<T *>(t.dst) + j * t.sd_col + head * t.sd_head;
        if (h + step < h1) load(h + step);
        if (HALF) {
            store4(d + lo, ya);
            store4(d + hi, yb);
        } else {
            const float y0[4] = {ya[0], yb[0], ya[1], yb[1]}, y1[4] = {ya[2], yb[2], ya[3], yb[3]};
            store4(d + lo, y0);
            store4(d + hi, y1);
        }
    }
}

template <typename T> cudaError_t launch_rope(RopeParams &p, int ncols, cudaStream_t s) {
    const int half = p.n_rot / 2, rest = p.head_dim - p.n_rot, groups = half / 4 + rest / 8;
    bool vec = half % 4 == 0 && rest % 8 == 0 && groups > 0 && groups <= kThreads;
    p.heads = 0;
    for (int k = 0; k < p.ntensors; ++k) {
        const RopeTensor &t = p.t[k];
        p.heads += t.heads;
        vec = vec && aligned_to(t.x, 16) && t.sx_col % 4 == 0 && t.sx_head % 4 == 0 && aligned_to(t.dst, 4 * sizeof(T)) &&
              t.sd_col % 4 == 0 && t.sd_head % 4 == 0;
    }
    if (!vec) return launch_request(k_rope<T>, dim3(ncols), kThreads, 0, dim3(0), p, s);
    p.lanes = 1;
    while (p.lanes < groups) p.lanes *= 2;
    const int step = kThreads / p.lanes;
    // a block takes all heads where there are columns for every SM several times over (8192 columns: 56 us, 71 us with a
    // block per step), else one step of them (8 columns 2.1 us, 4.7 us with a block per column)
    p.heads_per_block = ncols >= 592 ? p.heads : step;
    while (p.heads / p.heads_per_block >= 65535) p.heads_per_block *= 2;  // (a grid's second dimension)
    const dim3 grid(ncols, (p.heads + p.heads_per_block - 1) / p.heads_per_block);
    return launch_request(p.layout == Q4K_ROPE_HALF ? k_rope_vec<T, true> : k_rope_vec<T, false>, grid, kThreads, 0, dim3(0), p, s);
}

// heads x ncols runs of dim values: apart when one of the two strides steps over the other's whole span.
bool runs_apart(int64_t heads, int64_t sh, int64_t ncols, int64_t sc, int64_t dim) {
    if (heads == 1) return ncols == 1 || sc >= dim;
    if (ncols == 1) return sh >= dim;
    return (sh >= dim && sc >= (heads - 1) * sh + dim) || (sc >= dim && sh >= (ncols - 1) * sc + dim);
}

// The values as runs along the larger stride (columns of heads, or heads of columns).
Runs runs_of(const void *p, int64_t heads, int64_t sh, int64_t ncols, int64_t sc, int64_t dim, int esz) {
    if (ncols > 1 && (heads == 1 || sc >= sh)) return {p, ((heads - 1) * sh + dim) * esz, sc * esz, ncols};
    return {p, ((ncols > 1 ? (ncols - 1) * sc : 0) + dim) * esz, sh * esz, heads};
}

}  // namespace

extern "C" int q4k_rope_multi(const q4k_rope_tensor *tensors, int ntensors, int ncols, int head_dim, int n_rot,
                              const int32_t *pos, int64_t stride_axis_pos, const double *inv_freq,
                              const int *sections, int n_axes, int order, int layout, float scale, int dst_type,
                              q4k_stream_t stream) {
    if (ntensors < 0 || ntensors > Q4K_MAX_ROPE_TENSORS)
        return request_fail(Q4K_EINVAL, "ntensors=%d outside 0..%d", ntensors, Q4K_MAX_ROPE_TENSORS);
    if (!extent_ok(ncols)) return request_fail(Q4K_EINVAL, "ncols=%d < 0", ncols);
    if (head_dim < 1 || head_dim > Q4K_MAX_ROPE_DIM)
        return request_fail(Q4K_EINVAL, "head_dim=%d outside 1..%d", head_dim, Q4K_MAX_ROPE_DIM);
    if (n_rot < 0 || n_rot > head_dim || n_rot % 2)
        return request_fail(Q4K_EINVAL, "n_rot=%d is not an even number in 0..head_dim=%d", n_rot, head_dim);
    if (n_axes < 1 || n_axes > Q4K_MAX_ROPE_AXES)
        return request_fail(Q4K_EINVAL, "n_axes=%d outside 1..%d", n_axes, Q4K_MAX_ROPE_AXES);
    if (order != Q4K_ROPE_BLOCKS && order != Q4K_ROPE_INTERLEAVED)
        return request_fail(Q4K_EINVAL, "order=%d is not a Q4K_ROPE_* order", order);
    if (layout != Q4K_ROPE_HALF && layout != Q4K_ROPE_ADJACENT)
        return request_fail(Q4K_EINVAL, "layout=%d is not a Q4K_ROPE_* layout", layout);
    if (dst_type != Q4K_TYPE_F32 && dst_type != Q4K_TYPE_F16 && dst_type != Q4K_TYPE_BF16)
        return request_fail(Q4K_EINVAL, "dst_type=%d is not F32, F16 or BF16", dst_type);
    if (sections == nullptr) return request_fail(Q4K_EINVAL, "null sections");
    RopeParams p = {};
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0 || sections[a] > Q4K_MAX_ROPE_DIM)
            return request_fail(Q4K_EINVAL, "sections[%d]=%d outside 0..%d", a, sections[a], Q4K_MAX_ROPE_DIM);
        p.sect[a] = sections[a];
        p.sect_sum += sections[a];
    }
    if (p.sect_sum == 0 && order == Q4K_ROPE_BLOCKS) return request_fail(Q4K_EINVAL, "sections are all 0");
    if (ncols > 0 && ntensors > 0) {
        if (tensors == nullptr) return request_fail(Q4K_EINVAL, "null tensors");
        if (n_rot > 0) {
            if (pos == nullptr || !aligned_to(pos, 4) || inv_freq == nullptr || !aligned_to(inv_freq, 8))
                return request_fail(Q4K_EINVAL, "pos or inv_freq null or misaligned");
            if (!in_stride_ok(stride_axis_pos, n_axes > 1 ? ncols : 0))
                return request_fail(Q4K_EINVAL, "stride_axis_pos=%lld < ncols", (long long)stride_axis_pos);
        }
    }
    const int dsz = dst_type == Q4K_TYPE_F32 ? 4 : 2;
    for (int k = 0; k < ntensors && ncols > 0; ++k) {
        const q4k_rope_tensor &t = tensors[k];
        if (t.heads < 0 || t.heads > kMaxExtent / Q4K_MAX_ROPE_DIM)
            return request_fail(Q4K_EINVAL, "tensor %d: heads=%d", k, t.heads);
        if (t.heads == 0) continue;
        if (t.x == nullptr || t.dst == nullptr || !aligned_to(t.x, 4) || !aligned_to(t.dst, dsz))
            return request_fail(Q4K_EINVAL, "tensor %d: x or dst null or misaligned", k);
        if (!stride_ok(t.stride_head_x, 0) || !stride_ok(t.stride_head_dst, 0) || !stride_ok(t.stride_col_x, 0) ||
            !stride_ok(t.stride_col_dst, 0))
            return request_fail(Q4K_EINVAL, "tensor %d: a stride is negative or too large", k);
        if (!runs_apart(t.heads, t.stride_head_dst, ncols, t.stride_col_dst, head_dim))
            return request_fail(Q4K_EINVAL, "tensor %d: dst's heads overlap (head stride %lld, column stride %lld)", k,
                                (long long)t.stride_head_dst, (long long)t.stride_col_dst);
        p.t[p.ntensors++] = {t.x, t.dst, t.stride_col_x, t.stride_head_x, t.stride_col_dst, t.stride_head_dst, t.heads};
    }
    if (ncols == 0 || p.ntensors == 0) return Q4K_OK;
    // no dst may share a value with another dst or with an x, but for an x turned in place
    for (int i = 0; i < p.ntensors; ++i) {
        const RopeTensor &w = p.t[i];
        const Runs wr = runs_of(w.dst, w.heads, w.sd_head, ncols, w.sd_col, head_dim, dsz);
        for (int k = 0; k < p.ntensors; ++k) {
            const RopeTensor &r = p.t[k];
            const bool in_place = k == i && w.dst == r.x && dsz == 4 && (r.heads == 1 || w.sd_head == r.sx_head) &&
                                  (ncols == 1 || w.sd_col == r.sx_col);
            if (!in_place && runs_overlap(wr, runs_of(r.x, r.heads, r.sx_head, ncols, r.sx_col, head_dim, 4)))
                return request_fail(Q4K_EINVAL, "a dst overlaps an x it does not turn in place");
            if (k != i && runs_overlap(wr, runs_of(r.dst, r.heads, r.sd_head, ncols, r.sd_col, head_dim, dsz)))
                return request_fail(Q4K_EINVAL, "two dst overlap");
        }
    }
    p.pos = pos;
    p.inv_freq = inv_freq;
    p.sp_axis = stride_axis_pos;
    p.head_dim = head_dim;
    p.n_rot = n_rot;
    p.n_axes = n_axes;
    p.order = order;
    p.layout = layout;
    p.scale = scale;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = dst_type == Q4K_TYPE_F32   ? launch_rope<float>(p, ncols, s)
                          : dst_type == Q4K_TYPE_F16 ? launch_rope<__half>(p, ncols, s)
                                                     : launch_rope<__nv_bfloat16>(p, ncols, s);
    if (e != cudaSuccess) return request_cuda_fail(e, "rope launch");
    return Q4K_OK;
}
