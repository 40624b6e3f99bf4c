// What the paged cache's kernels share.
#pragma once

#include <cuda_bf16.h>

#include "kvc_common.cuh"

struct kvc_div { uint32_t magic, shift; };      // n / d by a divisor that the host knows, 0 <= n < 2^31, 1 <= d <= 2^31

static inline kvc_div kvc_make_div(uint32_t d) {
    kvc_div r;
    r.shift = 0;
    while ((1ull << r.shift) < d) r.shift++;
    r.magic = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - d)) / d + 1);
    return r;
}
__device__ __forceinline__ int kvc_divide(int n, const kvc_div &d) { return (int)((__umulhi(d.magic, (uint32_t)n) + (uint32_t)n) >> d.shift); }

constexpr int KVC_MAX_PAGE = 1 << 20;           // tokens of a page
