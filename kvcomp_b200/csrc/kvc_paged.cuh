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
