// q4k_logits.cu -- q4k_logits_process: penalties for repeated tokens, biases
// and masks on the head's logits, the greedy token and the log-sum-exp of the
// result, in one pass.
#include "q4k_device.cuh"
#include "q4k_request.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstddef>
#include <type_traits>

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
    int slots;  // listed tokens a CTA has room for
};

constexpr int kThreads = 256;
constexpr int kQuads = 4;                         // groups of 4 tokens per thread and chunk (at most 8)
constexpr int kChunk = kThreads * kQuads * 4;     // tokens in flight per CTA
constexpr int kSegment = 65536;                   // tokens whose listed places are held at a time
constexpr int kMinSlots = 256, kMaxSlots = 4096;  // listed tokens with room for their count and bias sum
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

// The listed tokens of one segment of a CTA's slice: a bit per token, the
// number of bits before each word, and a slot {token, count, number of biases,
// bias sum} per listed token, found by its rank among them.
struct Lists {
    uint32_t touched[kSegment / 32];
    uint16_t before[kSegment / 32];
    uint32_t sums[kThreads / 32];
    int repeats;           // whether a token has several biases
    int token[kMaxSlots];  // `slots` of them, then as many of the others: the launch sizes the memory
};

// What a CTA knows of its column's lists: history entries [0, nh), bias entries
// [b0, b1), each thread's first ones in registers.
struct Column {
    const int32_t *history;
    int nh, b0, b1;
    int htok[kAhead], btok[kAhead];
    float bval[kAhead];
};

// f(token) for every history entry, g(token, value) for every bias entry, in no order.
template <typename F, typename G>
__device__ __forceinline__ void for_lists(const LogitsParams &P, const Column &C, F f, G g) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f(C.htok[i]);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) g(C.btok[i], C.bval[i]);
    for (int e0 = kAhead * kThreads + tid; e0 < C.nh; e0 += kAhead * kThreads) {
        int tok[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) tok[i] = e0 + i * kThreads < C.nh ? C.history[e0 + i * kThreads] : -1;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f(tok[i]);
    }
    for (int e = C.b0 + kAhead * kThreads + tid; e < C.b1; e += kThreads) g(P.bias_tokens[e], P.bias_values[e]);
}

// Finds the listed ones of the tokens [base, base + n): counts (integer
// atomics: any order gives the same) and bias sums (in list order where a token
// has several). Returns how many there are; with more than `slots` nothing is
// summed.
__device__ __forceinline__ int scan_lists(const LogitsParams &P, const Column &C, Lists &S, int base, int n) {
    const int tid = threadIdx.x, lane = tid & 31, words = (n + 31) / 32, slots = P.slots;
    int *count = S.token + slots, *biases = count + slots;
    float *bias = reinterpret_cast<float *>(biases + slots);
    for (int i = tid; i < words; i += kThreads) S.touched[i] = 0u;
    if (tid == 0) S.repeats = 0;
    __syncthreads();
    // (base + n is at most the vocabulary; base can be below 0, where tok - base would overflow for the largest tok)
    auto in = [&](int tok) { return tok >= 0 && tok >= base && tok < base + n; };
    auto mark = [&](int tok) {
        if (in(tok)) atomicOr(&S.touched[(tok - base) >> 5], 1u << ((tok - base) & 31));
    };
    for_lists(P, C, mark, [&](int tok, float) { mark(tok); });
    __syncthreads();
    // a thread ranks a run of words
    const int run = (words + kThreads - 1) / kThreads, w0 = tid * run, w1 = min(words, w0 + run);
    uint32_t mine = 0;
    for (int w = w0; w < w1; ++w) mine += __popc(S.touched[w]);
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) S.sums[tid / 32] = upto;
    __syncthreads();
    uint32_t total = 0, at = upto - mine;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < tid / 32) at += S.sums[w];
        total += S.sums[w];
    }
    if (static_cast<int>(total) > slots) return static_cast<int>(total);
    for (int w = w0; w < w1; ++w) {
        S.before[w] = static_cast<uint16_t>(at);
        at += __popc(S.touched[w]);
    }
    for (int i = tid; i < static_cast<int>(total); i += kThreads) {
        count[i] = 0;
        biases[i] = 0;
        bias[i] = 0.0f;
    }
    __syncthreads();
    auto slot = [&](int tok) {
        const int i = tok - base;
        return S.before[i >> 5] + __popc(S.touched[i >> 5] & ((1u << (i & 31)) - 1u));
    };
    for_lists(
        P, C,
        [&](int tok) {
            if (!in(tok)) return;
            const int i = slot(tok);
            S.token[i] = tok;
            atomicAdd(&count[i], 1);
        },
        [&](int tok, float val) {
            if (!in(tok)) return;
            const int i = slot(tok);
            S.token[i] = tok;
            // (a token's only bias stays as it is stored here; of several, the sum below is formed anew)
            if (atomicAdd(&biases[i], 1) > 0)
                S.repeats = 1;
            else
                bias[i] = 0.0f + val;
        });
    __syncthreads();
    if (S.repeats && tid < 32) {  // one warp adds up the tokens with several biases, in list order
        for (int i = lane; i < static_cast<int>(total); i += 32)
            if (biases[i] > 1) bias[i] = 0.0f;
        __syncwarp();
        for (int e0 = C.b0; e0 < C.b1; e0 += 32) {
            const int tok = e0 + lane < C.b1 ? P.bias_tokens[e0 + lane] : -1;
            const float val = e0 + lane < C.b1 ? P.bias_values[e0 + lane] : 0.0f;
            const int i = in(tok) ? slot(tok) : -1;
            unsigned todo = __ballot_sync(0xffffffffu, i >= 0 && biases[max(i, 0)] > 1);
            for (; todo != 0; todo &= todo - 1) {
                if (lane == __ffs(todo) - 1) bias[i] += val;
                __syncwarp();
            }
        }
    }
    if (S.repeats) __syncthreads();
    return static_cast<int>(total);
}

// The ends of a row, token by token: values of the tokens of [0, v1) at v..v+3.
__device__ __forceinline__ float4 load_each(const float *l, int v, int v1) {
    return make_float4(v >= 0 && v < v1 ? l[v] : -INFINITY, v + 1 >= 0 && v + 1 < v1 ? l[v + 1] : -INFINITY,
                       v + 2 >= 0 && v + 2 < v1 ? l[v + 2] : -INFINITY, v + 3 >= 0 && v + 3 < v1 ? l[v + 3] : -INFINITY);
}
__device__ __noinline__ float4 load_end(const float *l, int v, int v1) { return load_each(l, v, v1); }
// Stores those tokens of z whose bit is set.
__device__ __forceinline__ void store_each(float *d, int v, float4 z, uint32_t bits) {
    if (bits & 1u) d[v] = z.x;
    if (bits & 2u) d[v + 1] = z.y;
    if (bits & 4u) d[v + 2] = z.z;
    if (bits & 8u) d[v + 3] = z.w;
}
// The terms of a quad's sum of exponentials around +inf: only infinite ones count, NaN stays.
__device__ __noinline__ float infinite_terms(float4 z) {
    auto term = [](float x) { return x == INFINITY ? 1.0f : x != x ? x : 0.0f; };
    return (term(z.x) + term(z.y)) + (term(z.z) + term(z.w));
}
// The bits of the tokens v..v+3 that lie in [0, v1).
__device__ __forceinline__ uint32_t of_row(int v, int v1) {
    return (v >= 0 ? 15u : 15u << -v) & (v + 4 <= v1 ? 15u : 15u >> (v + 4 - v1)) & 15u;
}

// A cluster per column; its CTAs split the vocabulary. A CTA first finds the
// listed tokens of its slice (segments of 65536 tokens: a bitmap, ranks, a
// slot per listed token), while its first logits are on their way; then a
// thread per slot finishes the listed tokens, and the warps stream all others
// without another barrier: kQuads loads of 16 bytes in flight per thread, every
// logit stored and taken into the statistics. (Finishing listed tokens inside
// the stream made every fourth quad of a warp wait for their chain of lookups.)
// The logits cross memory once in each direction, and those of quads that a
// mask forbids are not read. The CTAs' statistics meet in the
// first one's shared memory; the others leave without waiting.
// V4: rows of logits and dst are equally far from 16-byte boundaries, so four
// tokens go in one access; quads start on such a boundary (`shift` tokens
// before a multiple of 4), and only the quads at a row's ends go one by one.
// In a graph, 384 rows of 128257 logits: the pass alone 70 us (5.6 TB/s, 0.86
// of the measured copy rate; torch's copy of these unaligned rows takes 131),
// with token and log-sum-exp 77, with histories of up to 1024 85, all 99; one
// row of 32000: 2.1, 4.1, 5.1 and 6.4 us.
template <bool V4>
__global__ void __launch_bounds__(kThreads, 4) k_logits(const __grid_constant__ LogitsParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    Lists &S = *reinterpret_cast<Lists *>(smem);
    __shared__ Stat part[kThreads / 32], all[16];
    cg::cluster_group cluster = cg::this_cluster();
    const int nc = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
    const int64_t j = blockIdx.x / nc;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // (waited for below: every CTA has begun)
    pdl_launch_dependents();
    pdl_wait();
    const float *l = P.logits + j * P.s_col;
    float *d = P.dst + j * P.s_dst;
    // this CTA's tokens [v0, v1): whole quads of the row's alignment
    const int shift = V4 ? static_cast<int>(reinterpret_cast<uintptr_t>(l) / 4 % 4) : 0;
    const int quads = (P.nvocab + shift + 3) / 4, per = (quads + nc - 1) / nc;
    const int v0 = min(quads, me * per) * 4 - shift, v1 = min(P.nvocab, min(quads, me * per + per) * 4 - shift);
    const uint32_t *mask = nullptr;
    if (P.mask != nullptr) {
        const int64_t r = P.mask_rows != nullptr ? P.mask_rows[j] : j;
        if (r >= 0 && r < P.n_masks) mask = P.mask + r * P.s_mask;
    }
    Column C = {};
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (P.history != nullptr) {
        C.history = P.history + j * P.s_hist;
        C.nh = P.history_len != nullptr ? min(max(P.history_len[j], 0), P.max_history) : P.max_history;
        rep = P.penalties[3 * j];
        freq = P.penalties[3 * j + 1];
        pres = P.penalties[3 * j + 2];
    }
    if (P.bias_tokens != nullptr) {
        C.b0 = min(max(P.bias_offsets[j], 0), P.n_bias);
        C.b1 = min(max(P.bias_offsets[j + 1], C.b0), P.n_bias);
    }
    const bool lists = C.nh > 0 || C.b1 > C.b0, stats = P.token != nullptr || P.lse != nullptr;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        C.htok[i] = tid + i * kThreads < C.nh ? C.history[tid + i * kThreads] : -1;
        const int e = C.b0 + tid + i * kThreads;
        C.btok[i] = e < C.b1 ? P.bias_tokens[e] : -1;
        C.bval[i] = e < C.b1 ? P.bias_values[e] : 0.0f;
    }
    Stat st = {-INFINITY, 0.0f, INT_MAX};
    float4 z[kQuads];
    uint32_t allowed = ~0u;  // of the thread's quads, four bits each
    // asks for the quads of [base, v1) that are the thread's. full: all kChunk tokens are the CTA's (V4: and whole quads)
    auto load = [&](auto full, int base) {
        constexpr bool kFull = decltype(full)::value;
        if (mask != nullptr) {
            const int words = (P.nvocab + 31) / 32;
            allowed = 0u;
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                const int v = base + (q * kThreads + tid) * 4, lo = (kFull ? v : max(v, 0)) >> 5;
                const uint32_t w0 = kFull || lo < words ? mask[lo] : 0u;
                const uint32_t w1 = lo + 1 < words && (v & 31) > 28 ? mask[lo + 1] : 0u;
                allowed |= ((kFull || v >= 0 ? __funnelshift_r(w0, w1, v & 31) : w0 << -v) & 15u) << (4 * q);
            }
        }
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int v = base + (q * kThreads + tid) * 4;
            z[q] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if ((!kFull && v >= v1) || !(allowed >> (4 * q) & 15u)) continue;
            if (!V4)
                z[q] = load_each(l, v, v1);
            else if (kFull || (v >= 0 && v + 4 <= v1))
                z[q] = __ldcs(reinterpret_cast<const float4 *>(l + v));
            else
                z[q] = load_end(l, v, v1);
        }
    };
    auto is_full = [&](int base, int end) { return V4 && base >= 0 && base + kChunk <= end; };
    auto load_any = [&](int base) {
        if (is_full(base, v1))
            load(std::true_type(), base);
        else
            load(std::false_type(), base);
    };
    // finishes the loaded quads of [base, seg + n): all but the listed tokens
    auto finish = [&](auto full, int base, int seg, int n) {
        constexpr bool kFull = decltype(full)::value;
        float m = st.m, top[kQuads];
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int i = base - seg + (q * kThreads + tid) * 4, v = seg + i;
            top[q] = -INFINITY;
            if (!kFull && i >= n) continue;
            const uint32_t ok = allowed >> (4 * q) & 15u, listed = lists ? S.touched[i >> 5] >> (i & 31) & 15u : 0u;
            if (ok != 15u || listed != 0u) {
                const uint32_t out = ~ok | listed;
                if (out & 1u) z[q].x = -INFINITY;
                if (out & 2u) z[q].y = -INFINITY;
                if (out & 4u) z[q].z = -INFINITY;
                if (out & 8u) z[q].w = -INFINITY;
            }
            if (V4 && (kFull || (v >= 0 && v + 4 <= v1)) && listed == 0u)
                *reinterpret_cast<float4 *>(d + v) = z[q];
            else
                store_each(d, v, z[q], (kFull ? 15u : of_row(v, v1)) & ~listed);
            top[q] = fmaxf(fmaxf(z[q].x, z[q].y), fmaxf(z[q].z, z[q].w));  // (of numbers: NaN loses)
            m = fmaxf(m, top[q]);
        }
        if (!stats) return;
        // the chunk's maximum and its lowest quad, one rescaling of the sum, then the exponentials. -inf adds nothing
        // even while it is all that has been seen; NaN stays in the sum. The difference comes first: m log2(e) alone
        // would overflow for the largest values.
        if (m > st.m) {
            st.at = INT_MAX;
            st.s *= ex2((st.m - m) * kLog2e);
            st.m = m;
        }
        if (m > -INFINITY)
#pragma unroll
            for (int q = kQuads - 1; q >= 0; --q)
                if (top[q] == m) st.at = min(st.at, base + (q * kThreads + tid) * 4);
        const float around = m == -INFINITY ? 0.0f : m;
        if (m < INFINITY) {
#pragma unroll
            for (int q = 0; q < kQuads; ++q)
                if (kFull || base - seg + (q * kThreads + tid) * 4 < n)
                    st.s += (ex2((z[q].x - around) * kLog2e) + ex2((z[q].y - around) * kLog2e)) +
                            (ex2((z[q].z - around) * kLog2e) + ex2((z[q].w - around) * kLog2e));
        } else {
#pragma unroll
            for (int q = 0; q < kQuads; ++q)
                if (kFull || base - seg + (q * kThreads + tid) * 4 < n) st.s += infinite_terms(z[q]);
        }
    };
    int seg = v0, room = kSegment;
    if (v0 < v1) load_any(v0);
    while (seg < v1) {
        const int n = min(room, v1 - seg);
        if (lists) {
            const int total = scan_lists(P, C, S, seg, n);
            if (total > P.slots) {  // more than there are slots for: segments of as many tokens
                room = P.slots;
                __syncthreads();
                continue;
            }
            for (int i = tid; i < total; i += kThreads) {
                const int v = S.token[i], c = S.token[P.slots + i];
                float y = -INFINITY;
                if (mask == nullptr || (mask[v >> 5] >> (v & 31) & 1u)) {
                    y = __fadd_rn(l[v], __int_as_float(S.token[3 * P.slots + i]));
                    if (c > 0) {
                        y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                        y = __fsub_rn(y, __fadd_rn(__fmul_rn(static_cast<float>(c), freq), pres));
                    }
                }
                d[v] = y;
                // (NaN is never picked and stays in the sum)
                take(st, {y == y ? y : -INFINITY, y == -INFINITY ? 0.0f : y == y ? 1.0f : y, v - (v - v0) % 4});
            }
        }
        for (int base = seg; base < seg + n; base += kChunk) {
            if (is_full(base, seg + n))
                finish(std::true_type(), base, seg, n);
            else
                finish(std::false_type(), base, seg, n);
            const int next = base + kChunk < seg + n ? base + kChunk : seg + n;
            if (next < v1) load_any(next);
        }
        seg += n;
        if (lists && seg < v1) __syncthreads();  // the lists of this segment are done with
    }
    if (stats) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) take(st, shfl_xor(st, o));
        if (lane == 0) part[warp] = st;
        __syncthreads();
        if (warp == 0) {
            st = lane < kThreads / 32 ? part[lane] : Stat{-INFINITY, 0.0f, INT_MAX};
#pragma unroll
            for (int o = kThreads / 64; o > 0; o >>= 1) take(st, shfl_xor(st, o));
        }
    }
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (!stats) return;
    if (tid == 0) *cluster.map_shared_rank(all + me, 0) = st;
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (me != 0) return;
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 0) {
        st = lane < nc ? all[lane] : Stat{-INFINITY, 0.0f, INT_MAX};
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) take(st, shfl_xor(st, o));
        if (lane == 0) {
            if (P.token != nullptr) {
                int at = -1;
                if (st.m != -INFINITY)  // the quad holds it: its stored values say where
#pragma unroll
                    for (int e = 3; e >= 0; --e) {
                        const int v = st.at + e;
                        if (v >= 0 && v < P.nvocab && __ldcg(d + v) == st.m) at = v;
                    }
                P.token[j] = at;
            }
            if (P.lse != nullptr) P.lse[j] = st.s == 0.0f ? -INFINITY : (st.m == -INFINITY ? 0.0f : st.m) + logf(st.s);
        }
    }
}

size_t list_bytes(int slots) { return offsetof(Lists, token) + static_cast<size_t>(slots) * 16; }

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
                e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(list_bytes(kMaxSlots)));
            if (e != cudaSuccess) return e;
        }
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    // eight CTAs for every SM (four are resident: the rest evens out their ends) if the vocabulary has a chunk for each
    int nc = 1;
    while (nc < 16 && nc * kChunk < p.nvocab && nc * static_cast<int64_t>(ncols) < 1184) nc *= 2;
    // slots for a column's whole history and its likely biases (their number per column is known to the device
    // alone); a CTA whose tokens need more takes them in smaller segments, its whole slice from then on, and reads the
    // column's lists again for each: right, but slow for a column that holds most of a batch's biases
    const int64_t listed = p.max_history + (p.bias_tokens != nullptr ? 2 * static_cast<int64_t>(p.n_bias) / ncols + 64 : 0);
    LogitsParams q = p;
    q.slots = static_cast<int>(std::min<int64_t>(kMaxSlots, std::max<int64_t>(kMinSlots, (listed + 31) / 32 * 32)));
    const size_t smem = p.history != nullptr || p.bias_tokens != nullptr ? list_bytes(q.slots) : 0;
    return launch_request(fn, dim3(static_cast<unsigned>(ncols) * nc), kThreads, smem, dim3(nc), q, s);
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
