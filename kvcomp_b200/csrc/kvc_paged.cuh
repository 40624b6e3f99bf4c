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

__device__ __forceinline__ void raise_flag(int32_t *status, int flags) {
    if (flags && status) atomicOr(status, flags);
}

// ---- rotation
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float2 unpack(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ float2 unpack(uint32_t v, __nv_bfloat16) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v)); }
__device__ __forceinline__ uint32_t pack(float a, float b, __half) { const __half2 r = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&r); }
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) { const __nv_bfloat162 r = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&r); }

// cos and sin of a position, given the turns of one step.  The turns are counted in fp64: what is left of a far position's angle after its whole
// turns keeps 2^-53 of the angle, 1e-10 at a million radians; fp32 would keep 0.06.  Of the rest the nearest quarter is taken off, and the series of sine and cosine on
// [-pi / 4, pi / 4] are left, to x^9 and x^10: the first terms left out are below 2^-29 and 2^-33 (fp32's half step there: 2^-25).
constexpr double TURNS_OF_RADIANS = 0.15915494309189533576888;
__device__ __forceinline__ float2 turn_by(float x, int q, float factor) {
    const float y = x * x;
    float s = fmaf(y, 1.0f / 362880, -1.0f / 5040), c = fmaf(y, -1.0f / 3628800, 1.0f / 40320);
    s = fmaf(y, s, 1.0f / 120);
    c = fmaf(y, c, -1.0f / 720);
    s = fmaf(y, s, -1.0f / 6);
    c = fmaf(y, c, 1.0f / 24);
    s = fmaf(x * y, s, x);
    c = fmaf(y, c, -0.5f);
    c = fmaf(y, c, 1.0f);
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;
    return make_float2(((q + 1) & 2 ? -a : a) * factor, (q & 2 ? -b : b) * factor);
}
__device__ __forceinline__ float2 turn(double position, double turns, float factor) {
    double whole = position * turns;
    whole -= rint(whole);
    const float t = (float)whole, quarter = rintf(4.0f * t);
    return turn_by(fmaf(-0.25f, quarter, t) * 6.2831853071795865f, (int)quarter, factor);
}
// The same with the rest of a quarter taken in fp64 too: it is off by 2^-26, not by pi 2^-25 (the turn's own rounding), and cos and sin by little more than their last bit.  For keys that are
// coded next, of which what lies at the border of two codes is decided by that.
__device__ __forceinline__ float2 turn_closely(double position, double turns, float factor) {
    double whole = position * turns;
    whole -= rint(whole);
    const float quarter = rintf(4.0f * (float)whole);
    return turn_by((float)((whole - 0.25 * (double)quarter) * 6.283185307179586476925), (int)quarter, factor);
}

// Queries, keys or values: a CTA has rows of one of them.  dst: token stride 0 for the pools, where `places` say where a token goes.
struct Part {
    const void *src;
    void *dst;
    int64_t src_token, src_head, dst_token, dst_head;
    int heads, chunk, of_token, turned;                     // heads, those that a thread takes, threads' shares of a token, rotated units of a head
    unsigned first;                                         // CTA
    kvc_div chunks;                                         // by of_token
};
