// Attention of one new token per request over a paged key-value cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m) with s_t = scaling * q . k_t: one pass over the tokens with a running maximum m
// and a running sum l; whenever the maximum grows, sum and accumulators are multiplied with exp(m_old - m_new).
#include <cuda_bf16.h>
#include <math_constants.h>
#include <string.h>

#include "kvc_common.cuh"

namespace {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

constexpr int WARPS = 4;

// A CTA per (request, query head); its warps take every fourth token, a lane has D / 32 channels.
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) paged_attn_kernel(const kvc_paged_attn_args a) {
    constexpr int E = D / 32;
    __shared__ float acc_s[WARPS][D], m_s[WARPS], l_s[WARPS];
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int hk = h / (int)(a.Hq / a.Hkv);
    long long len = a.lengths[b];
    if (len < 0 || len > a.table_width * a.page_size) {
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, KVC_FLAG_BAD_LENGTH);
        len = len < 0 ? 0 : a.table_width * a.page_size;
    }
    const long long first = a.window > 0 && len > a.window ? len - a.window : 0;
    float q[E], acc[E] = {}, m = -CUDART_INF_F, l = 0.0f;
    for (int e = 0; e < E; e++) q[e] = to_float(reinterpret_cast<const T *>(a.q)[b * a.q_token + h * a.q_head + e * 32 + lane]);
    for (long long t = first + warp; t < len; t += WARPS) {
        const int page = a.table[b * a.table_stride + t / a.page_size];
        if ((unsigned)page >= (unsigned long long)a.n_pages) {
            if (lane == 0 && a.status) atomicOr(a.status, KVC_FLAG_BAD_PAGE);
            continue;
        }
        const T *k = reinterpret_cast<const T *>(a.kpages) + page * a.kp_page + t % a.page_size * a.kp_row + hk * a.kp_head;
        const T *v = reinterpret_cast<const T *>(a.vpages) + page * a.vp_page + t % a.page_size * a.vp_row + hk * a.vp_head;
        float s = 0.0f;
        for (int e = 0; e < E; e++) s += q[e] * to_float(k[e * 32 + lane]);
        s = kvc_warp_sum(s) * a.scaling;
        const float m_new = fmaxf(m, s), scale = m_new == -CUDART_INF_F ? 1.0f : __expf(m - m_new), p = m_new == -CUDART_INF_F ? 0.0f : __expf(s - m_new);
        m = m_new;
        l = l * scale + p;
        for (int e = 0; e < E; e++) acc[e] = acc[e] * scale + p * to_float(v[e * 32 + lane]);
    }
    for (int e = 0; e < E; e++) acc_s[warp][e * 32 + lane] = acc[e];
    if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
    __syncthreads();
    float top = -CUDART_INF_F, sum = 0.0f;
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, m_s[w]);
    for (int w = 0; w < WARPS; w++) sum += m_s[w] == -CUDART_INF_F ? 0.0f : l_s[w] * __expf(m_s[w] - top);
    for (int d = threadIdx.x; d < D; d += WARPS * 32) {
        float o = 0.0f;
        for (int w = 0; w < WARPS; w++) o += m_s[w] == -CUDART_INF_F ? 0.0f : acc_s[w][d] * __expf(m_s[w] - top);
        reinterpret_cast<T *>(a.out)[b * a.out_token + h * a.out_head + d] = from_float<T>(sum == 0.0f ? 0.0f : o / sum);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[b * a.Hq + h] = sum == 0.0f ? -CUDART_INF_F : top + logf(sum);
}

}  // namespace

extern "C" int64_t kvc_paged_attn_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    if (B < 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
    return 256;
}

extern "C" int kvc_paged_attn(const kvc_paged_attn_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_paged_attn: null pointer");
    kvc_paged_attn_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_paged_attn: unknown type %d", a.type);
    KVC_REQUIRE(a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256, "kvc_paged_attn: heads of 64, 96, 128 or 256 channels, got %lld", (long long)a.D);
    KVC_REQUIRE(a.B >= 0 && a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0 && a.Hq < 65536, "kvc_paged_attn: %lld query heads over %lld", (long long)a.Hq, (long long)a.Hkv);
    KVC_REQUIRE(a.page_size > 0 && a.page_size <= (1 << 20) && a.n_pages >= 0 && a.n_pages < (1ll << 31) && a.table_width >= 0 && a.window >= 0, "kvc_paged_attn: bad sizes");
    KVC_REQUIRE(a.table_width * a.page_size < (1ll << 31), "kvc_paged_attn: a table row holds %lld tokens, lengths have 32 bits", (long long)(a.table_width * a.page_size));
    if (a.B == 0) return KVC_OK;
    KVC_REQUIRE(a.B < 65536, "kvc_paged_attn: %lld requests", (long long)a.B);
    KVC_REQUIRE(a.q && a.out && a.lengths && (a.table || a.table_width == 0) && ((a.kpages && a.vpages) || a.n_pages == 0), "kvc_paged_attn: null pointer");
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages) | reinterpret_cast<uintptr_t>(a.out);
    if (a.Hq == 1) a.q_head = a.out_head = 0;              // (the stride of a dimension of one may be anything)
    if (a.B == 1) a.q_token = a.out_token = 0;
    if (a.Hkv == 1) a.kp_head = a.vp_head = 0;
    if (a.page_size == 1) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1) a.kp_page = a.vp_page = 0;
    const int64_t strides = a.q_token | a.q_head | a.out_token | a.out_head | a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head;
    KVC_REQUIRE((at & 15) == 0 && (strides & 7) == 0, "kvc_paged_attn: rows must start on 16 bytes");
    KVC_REQUIRE(a.workspace && (reinterpret_cast<uintptr_t>(a.workspace) & 15) == 0, "kvc_paged_attn: the workspace must be 16-byte aligned");
    if (a.workspace_bytes < kvc_paged_attn_workspace(a.B, a.Hq, a.Hkv, a.D)) {
        kvc_set_error("kvc_paged_attn: the workspace must hold what kvc_paged_attn_workspace says");
        return KVC_ERR_CAPACITY;
    }
    const dim3 grid((unsigned)a.Hq, (unsigned)a.B);
#define KVC_PA(T_, D_) paged_attn_kernel<T_, D_><<<grid, WARPS * 32, 0, kvc_cu(stream)>>>(a)
    if (a.type == KVC_TYPE_FP16) {
        if (a.D == 64) KVC_PA(__half, 64); else if (a.D == 96) KVC_PA(__half, 96); else if (a.D == 128) KVC_PA(__half, 128); else KVC_PA(__half, 256);
    } else {
        if (a.D == 64) KVC_PA(__nv_bfloat16, 64); else if (a.D == 96) KVC_PA(__nv_bfloat16, 96); else if (a.D == 128) KVC_PA(__nv_bfloat16, 128); else KVC_PA(__nv_bfloat16, 256);
    }
#undef KVC_PA
    KVC_LAUNCH_OK();
    return KVC_OK;
}
