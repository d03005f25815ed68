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
#ifndef LG_T
#define LG_T 256
#define LG_Q 4
#define LG_MB 4
#endif
constexpr int kThreads = LG_T;
constexpr int kQuads = LG_Q;                      // groups of 4 tokens per thread and chunk
constexpr int kChunk = kThreads * kQuads * 4;     // tokens whose counts and bias sums are in shared memory at a time
constexpr int kAhead = 4;                         // list entries per thread in registers
constexpr float kLog2e = 1.4426950408889634f;

// Running maximum, the first token of its (lowest) quad, and the sum of
// exponentials around it.
struct Stat {
    float m, s;
    int at;
};
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void take(Stat &a, const Stat &b) {
    const bool better = b.m > a.m || (b.m == a.m && b.at < a.at);
    const float m = better ? b.m : a.m;
    // (-inf: nothing seen yet; +inf: only the infinite terms count)
    const float ea = a.m == m ? 1.0f : ex2((a.m - m) * kLog2e), eb = b.m == m ? 1.0f : ex2((b.m - m) * kLog2e);
    a.s = m == -INFINITY ? a.s + b.s : a.s * ea + b.s * eb;
    if (better) a.at = b.at;
    a.m = m;
}
__device__ __forceinline__ Stat shfl_xor(const Stat &v, int o) {
    return {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
            __shfl_xor_sync(0xffffffffu, v.at, o)};
}

// Counts and bias sums of the listed tokens of one chunk. `touched` says which
// places hold something; the others are zero throughout.
struct Lists {
    int count[kChunk];
    float bias[kChunk];
    uint32_t touched[kChunk / 32];
};

// One warp adds 32 bias entries (lane order = list order) to the sums of the
// chunk [base, base + n); entries outside it are left out.
__device__ __forceinline__ void add_bias(Lists &S, int tok, float val, int base, int n, int lane) {
    const bool in = tok >= 0 && tok >= base && tok - base < n;
    if (!__any_sync(0xffffffffu, in)) return;
    const int i = in ? tok - base : 0;
    const unsigned same = __match_any_sync(0xffffffffu, in ? i : -1 - lane);
    if (in) atomicOr(&S.touched[i >> 5], 1u << (i & 31));
    if (__any_sync(0xffffffffu, __popc(same) > 1)) {
        for (int q = 0; q < 32; ++q) {  // a token twice: one entry after the other
            if (lane == q && in) S.bias[i] += val;
            __syncwarp();
        }
    } else if (in) {
        S.bias[i] += val;
    }
    __syncwarp();
}

__device__ __forceinline__ void add_count(Lists &S, int tok, int base, int n) {
    if (tok >= 0 && tok >= base && tok - base < n) {
        const int i = tok - base;
        atomicOr(&S.touched[i >> 5], 1u << (i & 31));
        atomicAdd(&S.count[i], 1);
    }
}

// What a CTA knows of its column.
struct Column {
    const float *l;
    float *d;
    const uint32_t *mask;  // or NULL
    const int32_t *history;
    int nh, b0, b1;        // history entries; bias entries [b0, b1)
    float rep, freq, pres;
    int v1;                // end of the CTA's tokens
    int htok[kAhead], btok[kAhead];  // the lists' first entries
    float bval[kAhead];
};

// Counts and bias sums of the chunk [base, base + n) from the column's lists.
__device__ __forceinline__ void scan_lists(const LogitsParams &P, const Column &C, Lists &S, int base, int n) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the bias entries go to the last warp, which has the fewest history entries
    if (warp == kThreads / 32 - 1) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (C.b0 + i * 32 < C.b1) add_bias(S, C.btok[i], C.bval[i], base, n, lane);
        for (int e0 = C.b0 + kAhead * 32; e0 < C.b1; e0 += kAhead * 32) {
            int tok[kAhead];
            float val[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int e = e0 + lane + i * 32;
                tok[i] = e < C.b1 ? P.bias_tokens[e] : -1;
                val[i] = e < C.b1 ? P.bias_values[e] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) add_bias(S, tok[i], val[i], base, n, lane);
        }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add_count(S, C.htok[i], base, n);
    for (int e0 = kAhead * kThreads + tid; e0 < C.nh; e0 += kAhead * kThreads) {
        int tok[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) tok[i] = e0 + i * kThreads < C.nh ? C.history[e0 + i * kThreads] : -1;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) add_count(S, tok[i], base, n);
    }
}

// One chunk of tokens from `base` on. FULL: all kChunk tokens are the CTA's
// and quads are aligned (V4); otherwise tokens outside [0, v1) are left out one by one.
template <bool V4, bool FULL, bool MASKED>
__device__ __forceinline__ void chunk(const LogitsParams &P, const Column &C, Lists &S, bool lists, bool stats, int base,
                                      Stat &st) {
    const int tid = threadIdx.x;
    const int n = FULL ? kChunk : min(kChunk, C.v1 - base);
    float z[kQuads][4];
    uint32_t bits[kQuads];  // allowed tokens of the quad
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const int v = base + (q * kThreads + tid) * 4;
        uint32_t m = 15u;
        if (MASKED) {
            const int words = (P.nvocab + 31) / 32, lo = FULL ? v >> 5 : max(v, 0) >> 5;
            const uint32_t w0 = FULL || lo < words ? C.mask[lo] : 0u;
            const uint32_t w1 = lo + 1 < words && (v & 31) > 28 ? C.mask[lo + 1] : 0u;
            m = FULL || v >= 0 ? __funnelshift_r(w0, w1, v & 31) & 15u : (w0 << -v) & 15u;
        }
        if (!FULL)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < 0 || v + e >= C.v1) m &= ~(1u << e);
        bits[q] = m;
    }
    // a logit is read where a token of its quad is allowed
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const int v = base + (q * kThreads + tid) * 4;
        if (V4 && (FULL || (v >= 0 && v + 4 <= C.v1))) {
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (!MASKED || bits[q]) x = __ldcs(reinterpret_cast<const float4 *>(C.l + v));
            z[q][0] = x.x, z[q][1] = x.y, z[q][2] = x.z, z[q][3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[q][e] = (bits[q] >> e) & 1u ? C.l[v + e] : 0.0f;
        }
    }
    if (lists) {
        __syncthreads();  // the last chunk's places are zero again
        scan_lists(P, C, S, base, n);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int i = (q * kThreads + tid) * 4;
            const uint32_t hit = S.touched[i >> 5] >> (i & 31) & 15u;
            if (hit) {
                const float4 b = *reinterpret_cast<const float4 *>(S.bias + i);
                const int4 c = *reinterpret_cast<const int4 *>(S.count + i);
                const float bv[4] = {b.x, b.y, b.z, b.w};
                const int cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[q][e] = __fadd_rn(z[q][e], bv[e]);
                    if (cv[e] > 0) {
                        float y = z[q][e];
                        y = y > 0.0f ? __fdiv_rn(y, C.rep) : __fmul_rn(y, C.rep);
                        z[q][e] = __fsub_rn(y, __fadd_rn(__fmul_rn(static_cast<float>(cv[e]), C.freq), C.pres));
                    }
                }
                *reinterpret_cast<float4 *>(S.bias + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<int4 *>(S.count + i) = make_int4(0, 0, 0, 0);
                atomicAnd(&S.touched[i >> 5], ~(15u << (i & 31)));
            }
        }
    }
    float m = st.m, top[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const int v = base + (q * kThreads + tid) * 4;
        if (MASKED || !FULL)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!((bits[q] >> e) & 1u)) z[q][e] = -INFINITY;
        if (V4 && (FULL || (v >= 0 && v + 4 <= C.v1))) {
            *reinterpret_cast<float4 *>(C.d + v) = make_float4(z[q][0], z[q][1], z[q][2], z[q][3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e >= 0 && v + e < C.v1) C.d[v + e] = z[q][e];
        }
        top[q] = fmaxf(fmaxf(z[q][0], z[q][1]), fmaxf(z[q][2], z[q][3]));  // (of numbers: NaN loses)
        m = fmaxf(m, top[q]);
    }
    if (!stats) return;
    // the chunk's maximum and its lowest quad (a thread's quads ascend), one rescaling of the sum, then the
    // exponentials. -inf adds nothing even while it is all that has been seen; NaN stays in the sum.
    if (m > st.m) {
#pragma unroll
        for (int q = kQuads - 1; q >= 0; --q)
            if (top[q] == m) st.at = base + (q * kThreads + tid) * 4;
        st.s *= ex2((st.m - m) * kLog2e);
        st.m = m;
    }
    if (m == INFINITY) {
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.s += z[q][e] == m ? 1.0f : z[q][e] != z[q][e] ? z[q][e] : 0.0f;
        return;
    }
    // (the difference first: m log2(e) alone would overflow for the largest values)
    const float around = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int q = 0; q < kQuads; ++q)
        st.s += (ex2((z[q][0] - around) * kLog2e) + ex2((z[q][1] - around) * kLog2e)) +
                (ex2((z[q][2] - around) * kLog2e) + ex2((z[q][3] - around) * kLog2e));
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
__global__ void __launch_bounds__(kThreads, LG_MB) k_logits(const __grid_constant__ LogitsParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    Lists &S = *reinterpret_cast<Lists *>(smem);
    __shared__ Stat part[kThreads / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const int nc = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
    const int64_t j = blockIdx.x / nc;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Column C;
    C.l = P.logits + j * P.s_col;
    C.d = P.dst + j * P.s_dst;
    // this CTA's tokens [v0, v1): whole quads of the row's alignment
    const int shift = V4 ? static_cast<int>(reinterpret_cast<uintptr_t>(C.l) / 4 % 4) : 0;
    const int quads = (P.nvocab + shift + 3) / 4, per = (quads + nc - 1) / nc;
    const int v0 = min(quads, me * per) * 4 - shift;
    C.v1 = min(P.nvocab, min(quads, me * per + per) * 4 - shift);
    C.nh = C.b0 = C.b1 = 0;
    C.rep = 1.0f;
    C.freq = C.pres = 0.0f;
    C.mask = nullptr;
    C.history = nullptr;
    if (P.history != nullptr) {
        C.history = P.history + j * P.s_hist;
        C.nh = P.history_len != nullptr ? min(max(P.history_len[j], 0), P.max_history) : P.max_history;
        C.rep = P.penalties[3 * j];
        C.freq = P.penalties[3 * j + 1];
        C.pres = P.penalties[3 * j + 2];
    }
    if (P.bias_tokens != nullptr) {
        C.b0 = min(max(P.bias_offsets[j], 0), P.n_bias);
        C.b1 = min(max(P.bias_offsets[j + 1], C.b0), P.n_bias);
    }
    if (P.mask != nullptr) {
        const int64_t r = P.mask_rows != nullptr ? P.mask_rows[j] : j;
        if (r >= 0 && r < P.n_masks) C.mask = P.mask + r * P.s_mask;
    }
    const bool lists = C.nh > 0 || C.b1 > C.b0, stats = P.token != nullptr || P.lse != nullptr;
    if (lists) {
        for (int i = tid; i < static_cast<int>(sizeof(Lists) / 16); i += kThreads)
            reinterpret_cast<int4 *>(&S)[i] = make_int4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            C.htok[i] = tid + i * kThreads < C.nh ? C.history[tid + i * kThreads] : -1;
            const int e = C.b0 + lane + i * 32;
            const bool mine = warp == kThreads / 32 - 1 && e < C.b1;
            C.btok[i] = mine ? P.bias_tokens[e] : -1;
            C.bval[i] = mine ? P.bias_values[e] : 0.0f;
        }
    }
    Stat st = {-INFINITY, 0.0f, INT_MAX};
    for (int base = v0; base < C.v1; base += kChunk) {
        if (V4 && base >= 0 && base + kChunk <= C.v1) {
            if (C.mask != nullptr)
                chunk<V4, V4, true>(P, C, S, lists, stats, base, st);
            else
                chunk<V4, V4, false>(P, C, S, lists, stats, base, st);
        } else {
            if (C.mask != nullptr)
                chunk<V4, false, true>(P, C, S, lists, stats, base, st);
            else
                chunk<V4, false, false>(P, C, S, lists, stats, base, st);
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
            if (P.token != nullptr) {
                int at = -1;
                if (st.m != -INFINITY)  // the quad holds it: its stored values say where
#pragma unroll
                    for (int e = 3; e >= 0; --e) {
                        const int v = st.at + e;
                        if (v >= 0 && v < P.nvocab && __ldcg(C.d + v) == st.m) at = v;
                    }
                P.token[j] = at;
            }
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
        for (auto *f : {k_logits<true>, k_logits<false>}) {
            e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Lists)));
            if (e != cudaSuccess) return e;
        }
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    int nc = 1;
    while (nc < 16 && nc * kChunk < p.nvocab && (LG_NC ? nc < LG_NC : nc * static_cast<int64_t>(ncols) < 4096)) nc *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ncols) * nc);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.history != nullptr || p.bias_tokens != nullptr ? sizeof(Lists) : 0;
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
