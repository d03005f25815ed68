// q4k_request.h -- host helpers shared by the entries that work on what each
// request of a batch brings of its own (q4k_lora.cu, q4k_rope.cu,
// q4k_logits.cu): error texts, address checks, launches.
#pragma once

#include "q4k_gemv.h"

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

namespace q4k {
void set_last_error_message(const char *msg);  // q4k_capi.cu

inline int request_fail(int status, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    set_last_error_message(buf);
    return status;
}

inline int request_cuda_fail(cudaError_t e, const char *what) {
    return request_fail(Q4K_ECUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

inline bool aligned_to(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Sizes and strides are kept where 64-bit byte offsets cannot overflow.
constexpr int64_t kMaxExtent = int64_t(1) << 30;
constexpr int64_t kMaxStride = int64_t(1) << 40;
inline bool extent_ok(int64_t v) { return v >= 0 && v <= kMaxExtent; }
inline bool stride_ok(int64_t v, int64_t least) { return v >= least && v <= kMaxStride; }
// Of an input's columns: 0 repeats one column.
inline bool in_stride_ok(int64_t v, int64_t least) { return v == 0 || stride_ok(v, least); }

// A strided set of byte runs: `count` runs of `len` bytes, `stride` bytes apart.
struct Runs {
    const void *p;
    int64_t len, stride, count;
};

// Whether two sets of runs share a byte.  Sets of one stride may interleave
// (slices of a fused buffer); for different strides, overlapping spans count
// as shared.
inline bool runs_overlap(const Runs &a, const Runs &b) {
    if (a.len <= 0 || b.len <= 0 || a.count <= 0 || b.count <= 0) return false;
    const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
    const intptr_t ea = pa + (a.count - 1) * a.stride + a.len, eb = pb + (b.count - 1) * b.stride + b.len;
    if (ea <= pb || eb <= pa) return false;
    if ((a.count == 1 && b.count == 1) || a.stride != b.stride || a.stride <= 0) return true;
    const intptr_t d = ((pb - pa) % a.stride + a.stride) % a.stride;  // offset of b's runs behind a's
    return d < a.len || a.stride - d < b.len;
}

// A launch that may begin while the one before it on the stream ends: its kernel
// waits for that one (griddepcontrol.wait) before it touches memory. cluster:
// 0 in x for none.
template <typename P>
cudaError_t launch_request(void (*fn)(P), dim3 grid, int threads, size_t smem, dim3 cluster, const P &p, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster.x;
    attr[1].val.clusterDim.y = cluster.y;
    attr[1].val.clusterDim.z = cluster.z;
    cfg.attrs = attr;
    cfg.numAttrs = cluster.x > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace q4k
