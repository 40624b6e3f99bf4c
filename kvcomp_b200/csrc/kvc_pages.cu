// Paged caches: which pages a step's tokens go to, the way back of finished requests' pages, and the rotation of queries and
// keys with the way of keys and values into their pages.
#include <cuda_bf16.h>
#include <string.h>

#include <algorithm>

#include "kvc_common.cuh"

namespace {

constexpr int SCAN_THREADS = 1024;
constexpr int MAX_PAGE = 1 << 20;

// ---- sums over the requests -----------------------------------------------------------------------------------

// exclusive sum of a and b over the CTA's threads, and the totals; every thread takes part
__device__ __forceinline__ void block_scan2(long long &a, long long &b, long long &total_a, long long &total_b, longlong2 *warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) { ia += ua; ib += ub; }
    }
    __syncthreads();                                        // (the sums of a scan before have been read)
    if (lane == 31) warps[warp] = make_longlong2(ia, ib);
    __syncthreads();
    long long fa = 0, fb = 0;
    total_a = total_b = 0;
    for (int w = 0; w < (int)blockDim.x / 32; w++) {
        const longlong2 v = warps[w];
        if (w < warp) { fa += v.x; fb += v.y; }
        total_a += v.x; total_b += v.y;
    }
    a = fa + ia - a;
    b = fb + ib - b;
}

__device__ __forceinline__ void raise_flag(int32_t *status, int flags) {
    if (flags && status) atomicOr(status, flags);
}

// the request whose rows hold `row`: the last b with starts[b] <= row among those that have any (starts[B] > row)
__device__ __forceinline__ int find_row(const int32_t *__restrict__ starts, int B, long long row) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(SCAN_THREADS) page_plan_kernel(const kvc_page_plan_args a) {
    __shared__ longlong2 warps[32];
    const int B = (int)a.B;
    const long long ps = a.page_size, head = min(max((long long)a.head[0], 0ll), (long long)a.n_pages);
    long long rows = 0, pages = 0, given = 0;              // in front of this thread's requests
    int flags = a.head[0] != head ? KVC_FLAG_BAD_LENGTH : 0;
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        long long held = 0, add = 0;
        if (b < B) { held = a.lengths[b]; add = a.new_tokens[b]; }
        if (held < 0 || add < 0) flags |= KVC_FLAG_BAD_LENGTH;
        held = held < 0 ? 0 : held; add = add < 0 ? 0 : add;
        long long start = add, zero = 0, total_rows, unused;
        block_scan2(start, zero, total_rows, unused, warps);
        start += rows;
        const long long owned = (held + ps - 1) / ps, wanted = (held + add + ps - 1) / ps;
        const bool fits = wanted <= a.table_width && start + add <= a.tokens && held + add < (1ll << 31);
        const long long need = fits ? wanted - owned : 0;
        long long before = need, total_need;
        block_scan2(before, zero, total_need, unused, warps);
        before += pages;
        const bool served = fits && (need == 0 || head + before + need <= a.n_pages);
        if (b < B) {
            a.starts[b] = (int32_t)min(start, (long long)a.tokens);
            a.taken[b] = served ? (int32_t)min(head + before, (long long)a.n_pages) : -1;
            a.lengths_out[b] = (int32_t)(served ? held + add : held);
            if (!served) flags |= KVC_FLAG_NO_PAGES;
        }
        if (served && need > 0) given = before + need;
        rows += total_rows; pages += total_need;
    }
    // the served that need pages are the first ones of those that need any: what they took is the largest sum
    long long best = given;
    __shared__ long long largest[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < SCAN_THREADS / 32; w++) best = max(best, largest[w]);
        a.starts[B] = (int32_t)min(rows, (long long)a.tokens);
        a.head_out[0] = (int32_t)(head + best);
    }
    raise_flag(a.status, flags);
    __threadfence_block();
    __syncthreads();
    const int end = a.starts[B];
    for (long long n = threadIdx.x; n < a.tokens; n += blockDim.x) {
        int slot = -1, position = 0;
        if (n < end) {
            const int b = find_row(a.starts, B, n), first = a.taken[b];
            const int add = max(a.new_tokens[b], 0), held = a.lengths_out[b] - (first >= 0 ? add : 0);
            position = held + (int)n - a.starts[b];
            if (first >= 0) {
                const int p = position / (int)ps, owned = (held + (int)ps - 1) / (int)ps;
                const int page = p >= owned ? a.free_pages[first + p - owned] : a.table[b * a.table_stride + p];
                if (p >= owned && position % (int)ps == 0) a.table[b * a.table_stride + p] = page;
                if ((unsigned)page < (unsigned long long)a.n_pages) slot = page * (int)ps + position % (int)ps;
                else raise_flag(a.status, KVC_FLAG_BAD_PAGE);
            }
        }
        a.slots[n] = slot;
        a.positions[n] = position;
    }
}

__global__ void __launch_bounds__(SCAN_THREADS) page_release_kernel(const kvc_page_release_args a) {
    __shared__ longlong2 warps[32];
    const int B = (int)a.B;
    const long long ps = a.page_size, head = min(max((long long)a.head[0], 0ll), (long long)a.n_pages);
    long long pages = 0, freed = 0;
    int flags = a.head[0] != head ? KVC_FLAG_BAD_LENGTH : 0;
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        const bool done = b < B && a.done[b] != 0;
        long long held = b < B ? a.lengths[b] : 0;
        if (held < 0 || (held + ps - 1) / ps > a.table_width) { flags |= KVC_FLAG_BAD_LENGTH; held = min(max(held, 0ll), ps * a.table_width); }
        const long long back = done ? (held + ps - 1) / ps : 0;
        long long before = back, zero = 0, total, unused;
        block_scan2(before, zero, total, unused, warps);
        before += pages;
        const bool fits = before + back <= head;
        if (done && !fits) flags |= KVC_FLAG_NO_PAGES;
        if (b < B) {
            a.first[b] = (int32_t)min(before, head);
            a.lengths_out[b] = done && fits ? 0 : (int32_t)held;
        }
        if (fits) freed = max(freed, before + back);
        pages += total;
    }
    __shared__ long long largest[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) freed = max(freed, __shfl_xor_sync(0xffffffffu, freed, o));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = freed;
    __syncthreads();
    for (int w = 0; w < SCAN_THREADS / 32; w++) freed = max(freed, largest[w]);
    if (threadIdx.x == 0) {
        a.first[B] = (int32_t)freed;
        a.head_out[0] = (int32_t)(head - freed);
    }
    raise_flag(a.status, flags);
    __threadfence_block();
    __syncthreads();
    for (long long i = threadIdx.x; i < freed; i += blockDim.x) {
        const int b = find_row(a.first, B, i);
        a.free_pages[head - freed + i] = a.table[b * a.table_stride + i - a.first[b]];
    }
}

// ---- rotation ---------------------------------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// cos and sin of position * frequency.  The turns are counted in fp64: what is left of a far position's angle after its whole
// turns keeps 2^-53 of the angle, 1e-10 at a million radians; fp32 would keep 0.06.
__device__ __forceinline__ float2 turn(int position, double frequency, float factor) {
    double t = (double)position * (frequency * 0.15915494309189533576888);
    t -= rint(t);
    float s, c;
    sincospif(2.0f * (float)t, &s, &c);
    return make_float2(c * factor, s * factor);
}

template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const kvc_rotary_args a) {
    const int half = (int)a.rotary / 2, units = (int)a.D - half;
    const long long heads = a.Hq + 2 * a.Hkv, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.N * heads * units) return;
    const int u = (int)(i % units);
    const int h = (int)(i / units % heads);
    const long long n = i / units / heads;
    const T *x;
    T *y;
    if (h < a.Hq) {
        x = reinterpret_cast<const T *>(a.q) + n * a.q_token + h * a.q_head;
        y = reinterpret_cast<T *>(a.q_out) + n * a.out_token + h * a.out_head;
    } else {
        const bool key = h < a.Hq + a.Hkv;
        const long long hk = h - a.Hq - (key ? 0 : a.Hkv);
        const int slot = a.slots[n];
        if (slot < 0) return;
        if (slot >= a.n_pages * a.page_size) { raise_flag(a.status, KVC_FLAG_BAD_PAGE); return; }
        const long long page = slot / a.page_size, row = slot % a.page_size;
        x = key ? reinterpret_cast<const T *>(a.k) + n * a.k_token + hk * a.k_head : reinterpret_cast<const T *>(a.v) + n * a.v_token + hk * a.v_head;
        y = key ? reinterpret_cast<T *>(a.kpages) + page * a.kp_page + row * a.kp_row + hk * a.kp_head
                : reinterpret_cast<T *>(a.vpages) + page * a.vp_page + row * a.vp_row + hk * a.vp_head;
    }
    if (u >= half) { y[half + u] = x[half + u]; return; }
    const int i0 = a.layout == KVC_ROTARY_HALF ? u : 2 * u, i1 = a.layout == KVC_ROTARY_HALF ? u + half : 2 * u + 1;
    const T x0 = x[i0], x1 = x[i1];
    if (h >= a.Hq + a.Hkv) { y[i0] = x0; y[i1] = x1; return; }
    float2 cs = turn(a.positions[n], a.frequencies[u], a.factor);
    if (a.inverse) cs.y = -cs.y;
    const float f0 = to_float(x0), f1 = to_float(x1);
    y[i0] = from_float<T>(f0 * cs.x - f1 * cs.y);
    y[i1] = from_float<T>(f1 * cs.x + f0 * cs.y);
}

}  // namespace

extern "C" int kvc_page_plan(const kvc_page_plan_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_page_plan: null pointer");
    kvc_page_plan_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.B >= 0 && a.B < (1 << 24) && a.n_pages >= 0 && a.page_size > 0 && a.page_size <= MAX_PAGE && a.tokens >= 0 && a.tokens < (1ll << 31),
                "kvc_page_plan: bad sizes");
    KVC_REQUIRE(a.n_pages * a.page_size < (1ll << 31), "kvc_page_plan: slots have 32 bits, the pool %lld tokens", (long long)(a.n_pages * a.page_size));
    KVC_REQUIRE(a.table_width >= 0 && a.table_width < (1ll << 31) && (a.B <= 1 || a.table_stride >= a.table_width), "kvc_page_plan: rows of the table overlap");
    KVC_REQUIRE(a.head && a.head_out && a.starts && (a.B == 0 || (a.lengths && a.new_tokens && a.lengths_out && a.taken)) && (a.free_pages || a.n_pages == 0) &&
                    (a.table || a.B == 0 || a.table_width == 0) && (a.tokens == 0 || (a.slots && a.positions)), "kvc_page_plan: null pointer");
    page_plan_kernel<<<1, SCAN_THREADS, 0, kvc_cu(stream)>>>(a);
    KVC_LAUNCH_OK();
    return KVC_OK;
}

extern "C" int kvc_page_release(const kvc_page_release_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_page_release: null pointer");
    kvc_page_release_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.B >= 0 && a.B < (1 << 24) && a.n_pages >= 0 && a.page_size > 0 && a.page_size <= MAX_PAGE && a.n_pages * a.page_size < (1ll << 31),
                "kvc_page_release: bad sizes");
    KVC_REQUIRE(a.table_width >= 0 && a.table_width < (1ll << 31) && (a.B <= 1 || a.table_stride >= a.table_width), "kvc_page_release: rows of the table overlap");
    KVC_REQUIRE(a.head && a.head_out && a.first && (a.B == 0 || (a.lengths && a.done && a.lengths_out)) && (a.free_pages || a.n_pages == 0) &&
                    (a.table || a.B == 0 || a.table_width == 0), "kvc_page_release: null pointer");
    page_release_kernel<<<1, SCAN_THREADS, 0, kvc_cu(stream)>>>(a);
    KVC_LAUNCH_OK();
    return KVC_OK;
}

extern "C" int kvc_rotary_store(const kvc_rotary_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_rotary_store: null pointer");
    kvc_rotary_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_rotary_store: unknown type %d", a.type);
    KVC_REQUIRE(a.layout == KVC_ROTARY_HALF || a.layout == KVC_ROTARY_INTERLEAVED, "kvc_rotary_store: unknown layout %d", a.layout);
    KVC_REQUIRE(a.N >= 0 && a.Hq >= 0 && a.Hkv >= 0 && a.D > 0 && a.D <= 65536 && a.rotary >= 0 && a.rotary <= a.D && a.rotary % 2 == 0,
                "kvc_rotary_store: bad sizes (head of %lld channels, %lld rotated)", (long long)a.D, (long long)a.rotary);
    KVC_REQUIRE(a.Hkv == 0 || (a.page_size > 0 && a.page_size <= MAX_PAGE && a.n_pages >= 0 && a.n_pages * a.page_size < (1ll << 31)), "kvc_rotary_store: bad pool");
    if (a.N == 0 || a.Hq + a.Hkv == 0) return KVC_OK;
    KVC_REQUIRE((a.Hq == 0 || (a.q && a.q_out)) && (a.Hkv == 0 || (a.k && a.v && a.slots && ((a.kpages && a.vpages) || a.n_pages == 0))) &&
                    (a.rotary == 0 || (a.positions && a.frequencies)), "kvc_rotary_store: null pointer");
    KVC_REQUIRE(a.Hq + 2 * a.Hkv < (1 << 20) && a.N < (1ll << 31), "kvc_rotary_store: too many heads or tokens");
    const long long n = a.N * (a.Hq + 2 * a.Hkv) * (a.D - a.rotary / 2);
    KVC_REQUIRE((n + 255) / 256 < (1ll << 31), "kvc_rotary_store: too many elements");
    auto *kernel = a.type == KVC_TYPE_FP16 ? rotary_kernel<__half> : rotary_kernel<__nv_bfloat16>;
    kernel<<<(unsigned)((n + 255) / 256), 256, 0, kvc_cu(stream)>>>(a);
    KVC_LAUNCH_OK();
    return KVC_OK;
}
