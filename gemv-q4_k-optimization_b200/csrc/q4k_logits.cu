// q4k_logits.cu -- q4k_logits_process: penalties for repeated tokens, biases
// and masks on the head's logits, the greedy token and the log-sum-exp of the
// result, in one pass.
#include "q4k_request.h"

#include <climits>

using namespace q4k;

namespace {

struct LogitsParams {
    const float *logits;
    float *dst;
    int64_t s_col, s_dst;
    const int32_t *history, *history_len;
    const float *penalties;
    int64_t s_hist;
    const int32_t *bias_tokens, *bias_offsets;
    const float *bias_values;
    const uint32_t *mask;
    const int32_t *mask_rows;
    int64_t s_mask;
    int32_t *token;
    float *lse;
    int nvocab, max_history, n_bias, n_masks;
};

constexpr int kThreads = 512;
constexpr int kChunk = 4096;  // tokens whose counts and bias sums are in shared memory at a time

// Running maximum (with its lowest index) and sum of exponentials around it.
struct Stat {
    float m, s;
    int at;
};
__device__ __forceinline__ float expo(float z, float m) { return exp2f((z - m) * 1.4426950408889634f); }
__device__ __forceinline__ void take(Stat &a, const Stat &b) {
    const bool better = b.m > a.m || (b.m == a.m && b.at < a.at);
    const float m = better ? b.m : a.m;
    // (-inf: nothing seen yet; +inf: only the infinite terms count)
    const float ea = a.m == m ? 1.0f : expo(a.m, m), eb = b.m == m ? 1.0f : expo(b.m, m);
    a.s = m == -INFINITY ? a.s + b.s : a.s * ea + b.s * eb;
    if (better) a.at = b.at;
    a.m = m;
}
__device__ __forceinline__ Stat stat_of(float z, int v) {
    if (z != z) return {-INFINITY, z, INT_MAX};  // NaN is never picked and stays in the sum
    if (z == -INFINITY) return {-INFINITY, 0.0f, INT_MAX};
    return {z, 1.0f, v};
}

// One CTA per column, chunk by chunk.
__global__ void __launch_bounds__(kThreads) k_logits(const __grid_constant__ LogitsParams P) {
    __shared__ int count[kChunk];
    __shared__ float bias[kChunk];
    __shared__ Stat part[kThreads / 32];
    const int64_t j = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *l = P.logits + j * P.s_col;
    float *d = P.dst + j * P.s_dst;
    int nh = 0, b0 = 0, b1 = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (P.history != nullptr) {
        nh = P.history_len != nullptr ? min(max(P.history_len[j], 0), P.max_history) : P.max_history;
        rep = P.penalties[3 * j];
        freq = P.penalties[3 * j + 1];
        pres = P.penalties[3 * j + 2];
    }
    if (P.bias_tokens != nullptr) {
        b0 = min(max(P.bias_offsets[j], 0), P.n_bias);
        b1 = min(max(P.bias_offsets[j + 1], b0), P.n_bias);
    }
    const uint32_t *mask = nullptr;
    if (P.mask != nullptr) {
        const int64_t r = P.mask_rows != nullptr ? P.mask_rows[j] : j;
        if (r >= 0 && r < P.n_masks) mask = P.mask + r * P.s_mask;
    }
    Stat st = {-INFINITY, 0.0f, INT_MAX};
    for (int base = 0; base < P.nvocab; base += kChunk) {
        const int n = min(kChunk, P.nvocab - base);
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            count[i] = 0;
            bias[i] = 0.0f;
        }
        __syncthreads();
        if (warp == 0) {  // bias entries in list order
            for (int e = b0; e < b1; e += 32) {
                const int tok = e + lane < b1 ? P.bias_tokens[e + lane] : -1;
                const bool in = tok >= base && tok - base < n;
                const int v = in ? tok - base : 0;
                if (!__any_sync(0xffffffffu, in)) continue;
                const float val = in ? P.bias_values[e + lane] : 0.0f;
                const unsigned same = __match_any_sync(0xffffffffu, in ? v : -1 - lane);
                if (__any_sync(0xffffffffu, __popc(same) > 1)) {
                    for (int q = 0; q < 32; ++q) {
                        if (lane == q && in) bias[v] += val;
                        __syncwarp();
                    }
                } else if (in) {
                    bias[v] += val;
                }
                __syncwarp();
            }
        } else {
            const int32_t *h = P.history + j * P.s_hist;
            for (int e = tid - 32; e < nh; e += kThreads - 32) {
                const int tok = h[e];
                if (tok >= base && tok - base < n) atomicAdd(&count[tok - base], 1);
            }
        }
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const int v = base + i;
            float z = l[v] + bias[i];
            if (count[i] > 0) {
                z = z > 0.0f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
                z = __fsub_rn(z, __fadd_rn(__fmul_rn(static_cast<float>(count[i]), freq), pres));
            }
            if (mask != nullptr && !((mask[v >> 5] >> (v & 31)) & 1u)) z = -INFINITY;
            d[v] = z;
            take(st, stat_of(z, v));
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        const Stat b = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                        __shfl_xor_sync(0xffffffffu, st.at, o)};
        take(st, b);
    }
    if (lane == 0) part[warp] = st;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 32; ++w) take(st, part[w]);
        if (P.token != nullptr) P.token[j] = st.m == -INFINITY ? -1 : st.at;
        if (P.lse != nullptr) P.lse[j] = st.s == 0.0f ? -INFINITY : (st.m == -INFINITY ? 0.0f : st.m) + logf(st.s);
    }
}

}  // namespace

extern "C" int q4k_logits_process(const q4k_logits_args *args, int ncols, q4k_stream_t stream) {
    if (args == nullptr) return request_fail(Q4K_EINVAL, "null args");
    const q4k_logits_args &a = *args;
    if (!extent_ok(ncols)) return request_fail(Q4K_EINVAL, "ncols=%d < 0", ncols);
    if (a.nvocab < 0 || a.nvocab > kMaxExtent) return request_fail(Q4K_EINVAL, "nvocab=%lld", (long long)a.nvocab);
    if (a.max_history < 0 || a.max_history > kMaxExtent)
        return request_fail(Q4K_EINVAL, "max_history=%lld", (long long)a.max_history);
    if (a.n_bias < 0 || a.n_bias > kMaxExtent) return request_fail(Q4K_EINVAL, "n_bias=%lld", (long long)a.n_bias);
    if (a.n_masks < 0) return request_fail(Q4K_EINVAL, "n_masks=%d < 0", a.n_masks);
    if (ncols == 0) return Q4K_OK;
    if (a.nvocab > 0 && (a.logits == nullptr || a.dst == nullptr || !aligned_to(a.logits, 4) || !aligned_to(a.dst, 4)))
        return request_fail(Q4K_EINVAL, "logits or dst null or misaligned");
    const int64_t least = ncols > 1 ? a.nvocab : 0;
    if (!in_stride_ok(a.stride_col, least) || !stride_ok(a.stride_col_dst, least))
        return request_fail(Q4K_EINVAL, "a column stride is below nvocab=%lld", (long long)a.nvocab);
    const bool in_place = a.logits == a.dst && (ncols == 1 || a.stride_col == a.stride_col_dst);
    if (!in_place && runs_overlap({a.logits, a.nvocab * 4, a.stride_col * 4, ncols},
                                  {a.dst, a.nvocab * 4, a.stride_col_dst * 4, ncols}))
        return request_fail(Q4K_EINVAL, "dst overlaps logits without being logits");
    const bool hist = a.max_history > 0 && (a.history != nullptr || a.penalties != nullptr);
    const bool bias = a.n_bias > 0;
    if (hist && (a.history == nullptr || a.penalties == nullptr))
        return request_fail(Q4K_EINVAL, "history and penalties go together");
    if (hist && !in_stride_ok(a.stride_history, ncols > 1 ? a.max_history : 0))
        return request_fail(Q4K_EINVAL, "stride_history=%lld < max_history", (long long)a.stride_history);
    if (bias && (a.bias_tokens == nullptr || a.bias_values == nullptr || a.bias_offsets == nullptr))
        return request_fail(Q4K_EINVAL, "bias_tokens, bias_values and bias_offsets go together");
    if (a.mask == nullptr && a.mask_rows != nullptr) return request_fail(Q4K_EINVAL, "mask_rows without a mask");
    if (a.mask != nullptr && !in_stride_ok(a.stride_mask, a.n_masks > 1 ? (a.nvocab + 31) / 32 : 0))
        return request_fail(Q4K_EINVAL, "stride_mask=%lld below nvocab/32", (long long)a.stride_mask);
    for (const void *p : {static_cast<const void *>(a.history), static_cast<const void *>(a.history_len),
                          static_cast<const void *>(a.penalties), static_cast<const void *>(a.bias_tokens),
                          static_cast<const void *>(a.bias_values), static_cast<const void *>(a.bias_offsets),
                          static_cast<const void *>(a.mask), static_cast<const void *>(a.mask_rows),
                          static_cast<const void *>(a.token), static_cast<const void *>(a.lse)})
        if (!aligned_to(p, 4)) return request_fail(Q4K_EINVAL, "a pointer is not 4-byte aligned");
    LogitsParams p = {};
    p.logits = a.logits;
    p.dst = a.dst;
    p.s_col = a.stride_col;
    p.s_dst = a.stride_col_dst;
    p.history = hist ? a.history : nullptr;
    p.history_len = a.history_len;
    p.penalties = a.penalties;
    p.s_hist = a.stride_history;
    p.bias_tokens = bias ? a.bias_tokens : nullptr;
    p.bias_offsets = a.bias_offsets;
    p.bias_values = a.bias_values;
    p.mask = a.n_masks > 0 ? a.mask : nullptr;
    p.mask_rows = a.mask_rows;
    p.s_mask = a.stride_mask;
    p.token = a.token;
    p.lse = a.lse;
    p.nvocab = static_cast<int>(a.nvocab);
    p.max_history = static_cast<int>(a.max_history);
    p.n_bias = static_cast<int>(a.n_bias);
    p.n_masks = a.n_masks;
    k_logits<<<ncols, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return request_cuda_fail(e, "logits launch");
    return Q4K_OK;
}
