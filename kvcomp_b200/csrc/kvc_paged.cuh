// What the paged cache's kernels share.
#pragma once

#include <cuda_bf16.h>

#include "kvc_common.cuh"

// n / d by a divisor that the host knows, 0 <= n < 2^31, 1 <= d <= 2^31: a product's high word, a sum and a shift (Granlund and Montgomery, Division by Invariant Integers using
// Multiplication, 1994)
struct kvc_div { uint32_t magic, shift; };

static inline kvc_div kvc_make_div(uint32_t d) {
    kvc_div r;
    r.shift = 0;
    while ((1ull << r.shift) < d) r.shift++;
    r.magic = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - d)) / d + 1);
    return r;
}
__device__ __forceinline__ int kvc_divide(int n, const kvc_div &d) { return (int)((__umulhi(d.magic, (uint32_t)n) + (uint32_t)n) >> d.shift); }

constexpr int KVC_MAX_PAGE = 1 << 20;           // tokens of a page

// ---- whether what a call writes overlaps (host)
// Rows of `width` bytes in up to three dimensions; those of size 1 are left out, and a stride of 0 says the same row again.  The others in the order of their strides, largest first.
struct kvc_rows {
    intptr_t at;
    int64_t width, size[3], stride[3], bytes;   // bytes: from the first to behind the last
    int dims, turned;                           // turned: a bit for each dimension whose stride was negative
    bool apart;                                 // each stride is at least what all smaller ones span
};
static inline kvc_rows kvc_make_rows(const void *at, int64_t width, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2 = 1, int64_t s2 = 0) {
    kvc_rows r = {reinterpret_cast<intptr_t>(at), 2 * width, {}, {}, 2 * width, 0, 0, true};
    const int64_t n[3] = {n0, n1, n2}, of[3] = {2 * s0, 2 * s1, 2 * s2};
    bool some = true;
    for (int i = 0; i < 3; i++) {
        int64_t s = of[i];
        some &= n[i] > 0;
        if (n[i] <= 1) continue;
        if (s == 0) { r.apart = false; continue; }
        if (s < 0) { r.at += (n[i] - 1) * s; r.turned |= 1 << i; s = -s; }
        int k = r.dims++;
        for (; k > 0 && r.stride[k - 1] < s; k--) { r.stride[k] = r.stride[k - 1]; r.size[k] = r.size[k - 1]; }
        r.stride[k] = s;
        r.size[k] = n[i];
    }
    for (int k = r.dims - 1; k >= 0; k--) {
        r.apart &= r.stride[k] >= r.bytes;
        r.bytes += (r.size[k] - 1) * r.stride[k];
    }
    if (!some) r.bytes = 0;
    return r;
}
static inline bool kvc_rows_equal(const kvc_rows &a, const kvc_rows &b) {
    bool same = a.at == b.at && a.dims == b.dims && a.turned == b.turned && a.apart == b.apart;
    for (int k = 0; k < a.dims && same; k++) same = a.stride[k] == b.stride[k] && a.size[k] == b.size[k];
    return same;
}
// Whether rows share memory: whether a difference of indices makes up for their distance.  From the largest stride of either on the quotient is that difference, or one of its
// neighbours, since what the smaller strides span is no more than it; where it is more (rows in and out of one another), the answer is yes.
static inline bool kvc_rows_overlap(const kvc_rows &a, const kvc_rows &b) {
    if (a.at + a.bytes <= b.at || b.at + b.bytes <= a.at) return false;
    int64_t stride[6], of_a[6], of_b[6], span_a = a.width, span_b = b.width;
    int dims = 0;
    for (int i = 0, j = 0; i < a.dims || j < b.dims; dims++) {
        const int64_t s = i == a.dims ? b.stride[j] : j == b.dims ? a.stride[i] : a.stride[i] > b.stride[j] ? a.stride[i] : b.stride[j];
        stride[dims] = s;
        of_a[dims] = i < a.dims && a.stride[i] == s ? a.size[i++] : 1;
        of_b[dims] = j < b.dims && b.stride[j] == s ? b.size[j++] : 1;
    }
    for (int k = dims - 1; k >= 0; k--) {
        if (span_a > stride[k] || span_b > stride[k]) return true;
        span_a += (of_a[k] - 1) * stride[k];
        span_b += (of_b[k] - 1) * stride[k];
    }
    struct { int64_t distance; int k; } left[16];           // (two differences at most leave less than a stride: one more entry for each of six levels)
    int n = 0;
    left[n++] = {b.at - a.at, 0};
    while (n > 0) {
        const auto now = left[--n];
        if (now.k == dims) {
            if (now.distance < a.width && -now.distance < b.width) return true;
            continue;
        }
        const int64_t s = stride[now.k], q = now.distance / s;
        for (int64_t d = q - 1; d <= q + 1; d++) {
            const int64_t rest = now.distance - d * s;
            if (d < of_a[now.k] && -d < of_b[now.k] && rest < s && -rest < s) left[n++] = {rest, now.k + 1};
        }
    }
    return false;
}

// A launch that may begin while the kernel ahead of it on the stream ends; every such kernel starts with kvc_behind().  (Not the attention's: the next launch's CTAs would
// take the places of those that have nothing to do, and its working ones lie unevenly: 8 x 4096 tokens of 32 heads 84.5 us, 96 so.)
template <typename P>
static inline int kvc_launch_early(void (*kernel)(const P), unsigned grid, unsigned threads, cudaStream_t stream, const P &p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    KVC_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p));
    return KVC_OK;
}
// Waits until all kernels ahead are done and what they wrote is seen; only then may the next kernel begin, so that it too finds everything ahead of this one done
// (a kernel that reads before it waits, as the compressed cache's attention does, relies on that).
__device__ __forceinline__ void kvc_behind() {
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
}
