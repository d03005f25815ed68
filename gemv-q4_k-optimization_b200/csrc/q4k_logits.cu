// q4k_logits.cu -- q4k_logits_process: penalties for repeated tokens, biases
// and masks on the head's logits, the greedy token and the log-sum-exp of the
// result, in one pass.
#include "q4k_request.h"

#include <cooperative_groups.h>

#include <atomic>
#include <climits>

using namespace q4k;
namespace cg = cooperative_groups;

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

#ifndef LG_NC
#define LG_NC 0
#endif
constexpr int kThreads = 256;
constexpr int kQuads = 4;                         // groups of 4 tokens per thread and chunk
constexpr int kChunk = kThreads * kQuads * 4;     // tokens whose counts and bias sums are in shared memory at a time

constexpr int kAhead = 4;                         // list entries per thread in registers
constexpr float kLog2e = 1.4426950408889634f;

// Running maximum (with its lowest index) and sum of exponentials around it.
struct Stat {
    float m, s;
    int at;
};
__device__ __forceinline__ float expo(float z, float m) { return exp2f((z - m) * kLog2e); }
__device__ __forceinline__ void take(Stat &a, const Stat &b) {
    const bool better = b.m > a.m || (b.m == a.m && b.at < a.at);
    const float m = better ? b.m : a.m;
    // (-inf: nothing seen yet; +inf: only the infinite terms count)
    const float ea = a.m == m ? 1.0f : expo(a.m, m), eb = b.m == m ? 1.0f : expo(b.m, m);
    a.s = m == -INFINITY ? a.s + b.s : a.s * ea + b.s * eb;
    if (better) a.at = b.at;
    a.m = m;
}
__device__ __forceinline__ Stat shfl_xor(const Stat &v, int o) {
    return {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
            __shfl_xor_sync(0xffffffffu, v.at, o)};
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One warp adds 32 bias entries (lane order = list order) to the sums of the
// chunk [base, base + n); entries outside it are left out.
__device__ __forceinline__ void add_bias(float *bias, int tok, float val, int base, int n, int lane) {
    const bool in = tok >= 0 && tok >= base && tok - base < n;
    if (!__any_sync(0xffffffffu, in)) return;
    const int i = in ? tok - base : 0;
    const unsigned same = __match_any_sync(0xffffffffu, in ? i : -1 - lane);
    if (__any_sync(0xffffffffu, __popc(same) > 1)) {
        for (int q = 0; q < 32; ++q) {  // a token twice: one entry after the other
            if (lane == q && in) bias[i] += val;
            __syncwarp();
        }
    } else if (in) {
        bias[i] += val;
    }
    __syncwarp();
}

__device__ __forceinline__ void add_count(int *count, int tok, int base, int n) {
    if (tok >= 0 && tok >= base && tok - base < n) atomicAdd(&count[tok - base], 1);
}

// A cluster per column; its CTAs split the vocabulary and walk their slices in
// chunks of kChunk tokens. Per chunk: the logits are asked for; the column's
// lists are scanned for tokens of the chunk, whose counts (integer atomics: any
// order gives the same) and bias sums (one warp, in list order) meet in shared
// memory; then every logit is finished in registers, stored, and taken into the
// running statistics. The logits cross memory once in each direction.
// V4: rows of logits and dst are equally far from 16-byte boundaries, so four
// tokens go in one access; chunks start on such a boundary (`shift` tokens
// before a multiple of 4), the ends of a row are handled one by one.
template <bool V4>
__global__ void __launch_bounds__(kThreads) k_logits(const __grid_constant__ LogitsParams P) {
    __shared__ __align__(16) int count[kChunk];
    __shared__ __align__(16) float bias[kChunk];
    __shared__ Stat part[kThreads / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const int nc = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
    const int64_t j = blockIdx.x / nc;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *l = P.logits + j * P.s_col;
    float *d = P.dst + j * P.s_dst;
    // this CTA's tokens [v0, v1): whole quads of the row's alignment
    const int shift = V4 ? static_cast<int>(reinterpret_cast<uintptr_t>(l) / 4 % 4) : 0;
    const int quads = (P.nvocab + shift + 3) / 4, per = (quads + nc - 1) / nc;
    const int v0 = min(quads, me * per) * 4 - shift, v1 = min(P.nvocab, min(quads, me * per + per) * 4 - shift);

    int nh = 0, b0 = 0, b1 = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    const uint32_t *mask = nullptr;
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
    if (P.mask != nullptr) {
        const int64_t r = P.mask_rows != nullptr ? P.mask_rows[j] : j;
        if (r >= 0 && r < P.n_masks) mask = P.mask + r * P.s_mask;
    }
    const bool lists = nh > 0 || b1 > b0, stats = P.token != nullptr || P.lse != nullptr;
    const int words = (P.nvocab + 31) / 32;
    Stat st = {-INFINITY, 0.0f, INT_MAX};
    if (lists)
        for (int i = tid; i < kChunk / 4; i += kThreads) {
            reinterpret_cast<int4 *>(count)[i] = make_int4(0, 0, 0, 0);
            reinterpret_cast<float4 *>(bias)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    // the first entries of the lists stay in registers over the chunks
    int htok[kAhead], btok[kAhead];
    float bval[kAhead];
    const int32_t *h = P.history + j * P.s_hist;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        htok[i] = tid + i * kThreads < nh ? h[tid + i * kThreads] : -1;
        const int e = b0 + lane + i * 32;
        btok[i] = warp == 0 && e < b1 ? P.bias_tokens[e] : -1;
        bval[i] = warp == 0 && e < b1 ? P.bias_values[e] : 0.0f;
    }
    for (int base = v0; base < v1; base += kChunk) {
        const int n = min(kChunk, v1 - base);
        // the chunk's allowed bits, then its logits where one is allowed
        float z[kQuads][4];
        uint32_t bits[kQuads];
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int v = base + (q * kThreads + tid) * 4;
            uint32_t m = 15u;
            if (mask != nullptr) {
                const int lo = max(v, 0) >> 5;
                const uint32_t w0 = lo < words ? mask[lo] : 0u, w1 = lo + 1 < words && (v & 31) > 28 ? mask[lo + 1] : 0u;
                m = v >= 0 ? __funnelshift_r(w0, w1, v & 31) : w0 << -v;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < 0 || v + e >= v1) m &= ~(1u << e);
            bits[q] = m & 15u;
        }
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int v = base + (q * kThreads + tid) * 4;
            if (V4 && v >= 0 && v + 4 <= v1) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (bits[q]) x = __ldcs(reinterpret_cast<const float4 *>(l + v));
                z[q][0] = x.x, z[q][1] = x.y, z[q][2] = x.z, z[q][3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[q][e] = (bits[q] >> e) & 1u ? l[v + e] : 0.0f;
            }
        }
        if (lists) {
            __syncthreads();  // zeros are in place
#pragma unroll
            for (int i = 0; i < kAhead; ++i) add_count(count, htok[i], base, n);
            for (int e0 = kAhead * kThreads + tid; e0 < nh; e0 += kAhead * kThreads) {
                int tok[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) tok[i] = e0 + i * kThreads < nh ? h[e0 + i * kThreads] : -1;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) add_count(count, tok[i], base, n);
            }
            if (warp == 0) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (b0 + i * 32 < b1) add_bias(bias, btok[i], bval[i], base, n, lane);
                for (int e0 = b0 + kAhead * 32; e0 < b1; e0 += kAhead * 32) {
                    int tok[kAhead];
                    float val[kAhead];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        const int e = e0 + lane + i * 32;
                        tok[i] = e < b1 ? P.bias_tokens[e] : -1;
                        val[i] = e < b1 ? P.bias_values[e] : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) add_bias(bias, tok[i], val[i], base, n, lane);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int i = (q * kThreads + tid) * 4, v = base + i;
            if (i >= n) continue;
            if (lists) {
                const float4 b = *reinterpret_cast<const float4 *>(bias + i);
                const int4 c = *reinterpret_cast<const int4 *>(count + i);
                const float bv[4] = {b.x, b.y, b.z, b.w};
                const int cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[q][e] = __fadd_rn(z[q][e], bv[e]);
                    if (cv[e] > 0) {
                        float y = z[q][e];
                        y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                        z[q][e] = __fsub_rn(y, __fadd_rn(__fmul_rn(static_cast<float>(cv[e]), freq), pres));
                    }
                }
                if (c.x | c.y | c.z | c.w) *reinterpret_cast<int4 *>(count + i) = make_int4(0, 0, 0, 0);
                // (any bits but zero, a NaN among them)
                if (__float_as_int(b.x) | __float_as_int(b.y) | __float_as_int(b.z) | __float_as_int(b.w))
                    *reinterpret_cast<float4 *>(bias + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!((bits[q] >> e) & 1u)) z[q][e] = -INFINITY;
            if (V4 && v >= 0 && v + 4 <= v1) {
                *reinterpret_cast<float4 *>(d + v) = make_float4(z[q][0], z[q][1], z[q][2], z[q][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v + e >= 0 && v + e < v1) d[v + e] = z[q][e];
            }
        }
        if (!stats) continue;
        // the chunk's maximum with its lowest index (a thread's tokens ascend), one rescaling of the sum, then
        // the exponentials. -inf adds nothing even while it is all that has been seen; NaN stays in the sum.
        float m = st.m;
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
            if ((q * kThreads + tid) * 4 < n) m = fmaxf(fmaxf(fmaxf(z[q][0], z[q][1]), fmaxf(z[q][2], z[q][3])), m);
        if (m > st.m) {
            int at = INT_MAX;
#pragma unroll
            for (int q = kQuads - 1; q >= 0; --q)
#pragma unroll
                for (int e = 3; e >= 0; --e)
                    if ((q * kThreads + tid) * 4 < n && z[q][e] == m) at = base + (q * kThreads + tid) * 4 + e;
            st.s *= expo(st.m, m);
            st.m = m;
            st.at = at;
        }
        const float around = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            if ((q * kThreads + tid) * 4 >= n) continue;
            if (m == INFINITY) {
#pragma unroll
                for (int e = 0; e < 4; ++e) st.s += z[q][e] == m ? 1.0f : z[q][e] != z[q][e] ? z[q][e] : 0.0f;
            } else {
                st.s += (ex2((z[q][0] - around) * kLog2e) + ex2((z[q][1] - around) * kLog2e)) +
                        (ex2((z[q][2] - around) * kLog2e) + ex2((z[q][3] - around) * kLog2e));
            }
        }
    }
    if (!stats) return;  // (the whole cluster)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) take(st, shfl_xor(st, o));
    if (lane == 0) part[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = lane < kThreads / 32 ? part[lane] : Stat{-INFINITY, 0.0f, INT_MAX};
#pragma unroll
        for (int o = kThreads / 64; o > 0; o >>= 1) take(st, shfl_xor(st, o));
        if (lane == 0) part[0] = st;
    }
    cluster.sync();
    if (me == 0 && warp == 0) {
        st = lane < nc ? cluster.map_shared_rank(part, lane)[0] : Stat{-INFINITY, 0.0f, INT_MAX};
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) take(st, shfl_xor(st, o));
        if (lane == 0) {
            if (P.token != nullptr) P.token[j] = st.m == -INFINITY ? -1 : st.at;
            if (P.lse != nullptr) P.lse[j] = st.s == 0.0f ? -INFINITY : (st.m == -INFINITY ? 0.0f : st.m) + logf(st.s);
        }
    }
    cluster.sync();  // no CTA leaves while another may still read its part
}

cudaError_t launch_logits(const LogitsParams &p, int ncols, cudaStream_t s) {
    const bool v4 = p.nvocab >= 16 && reinterpret_cast<uintptr_t>(p.logits) / 4 % 4 == reinterpret_cast<uintptr_t>(p.dst) / 4 % 4 &&
                    (ncols == 1 || p.s_col % 4 == p.s_dst % 4);
    auto *fn = v4 ? k_logits<true> : k_logits<false>;
    static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(k_logits<true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k_logits<false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    int nc = 1;
    while (nc < 16 && nc * kChunk < p.nvocab && (LG_NC ? nc < LG_NC : nc * static_cast<int64_t>(ncols) < 4096)) nc *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ncols) * nc);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nc;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, p);
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
    const cudaError_t e = launch_logits(p, ncols, reinterpret_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return request_cuda_fail(e, "logits launch");
    return Q4K_OK;
}
