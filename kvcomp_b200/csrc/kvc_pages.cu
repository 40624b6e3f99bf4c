// Paged caches: which pages a step's tokens go to, the way back of finished requests' pages, and the rotation of queries and
// keys with the way of keys and values into their pages.
#include <string.h>

#include <algorithm>

#include "kvc_paged.cuh"

namespace {

__device__ __forceinline__ void raise_flag(int32_t *status, int flags) {
    if (flags && status) atomicOr(status, flags);
}

// ---- pages ----------------------------------------------------------------------------------------------------------
//
// Two sums over the requests in their order (tokens, pages) say where each one's rows and pages begin; one CTA makes them, 1024
// requests at a time, since a launch for a step has little more to do than that.  What is left is 8 bytes for each token or page: where they are few the same CTA
// writes them behind a barrier, else a second kernel does, which reads what the first has written and never the lengths and the counter, so that
// these may be changed in place.  (All kernels of this file may begin while the one ahead ends, and wait for it: 131072 rows in two kernels 11.0 us a call, 9.6 so.)

constexpr int SCAN_THREADS = 1024, SMALL_THREADS = 128, FILL_THREADS = 256;
// Rows that the scanning CTA fills itself.  A second launch costs some 2 us, and so do 4096 rows of one CTA (16 a thread).
constexpr int FILL_ALONE = 4096;

// exclusive sums of a and b over the CTA's threads, and the totals; every thread takes part
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
    longlong2 v = lane < (int)blockDim.x / 32 ? warps[lane] : make_longlong2(0, 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ua = __shfl_up_sync(0xffffffffu, v.x, o), ub = __shfl_up_sync(0xffffffffu, v.y, o);
        if (lane >= o) { v.x += ua; v.y += ub; }
    }
    total_a = __shfl_sync(0xffffffffu, v.x, 31);
    total_b = __shfl_sync(0xffffffffu, v.y, 31);
    const long long fa = __shfl_sync(0xffffffffu, v.x, max(warp - 1, 0)), fb = __shfl_sync(0xffffffffu, v.y, max(warp - 1, 0));
    a = (warp ? fa : 0) + ia - a;
    b = (warp ? fb : 0) + ib - b;
}

__device__ __forceinline__ long long block_max(long long v, long long *warps) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 32; w++) v = max(v, warps[w]);
    return v;
}

// the request whose rows hold `row`: the last b with starts[b] <= row (behind it starts[b + 1] > row: it has some)
__device__ __forceinline__ int find_row(const int32_t *starts, int B, int row) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(int tokens, const kvc_div &page) { return tokens > 0 ? kvc_divide(tokens - 1, page) + 1 : 0; }

struct PlanParams { kvc_page_plan_args a; kvc_div page; };

// What rows are found by, where the request's threads left it: results in memory, or (held, the lengths before) the CTA's shared memory
struct Found { const int32_t *starts, *taken, *held; };

// slots and positions of rows [first, first + 4)
__device__ __forceinline__ void plan_rows(const PlanParams &p, const Found &f, int first, int end) {
    const kvc_page_plan_args &a = p.a;
    int slot[4], position[4];
    int b = -1, behind = 0, start = 0, taken = 0, held = 0, owned = 0, flags = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int n = first + k;
        slot[k] = -1;
        position[k] = 0;
        if (n >= end) continue;
        if (b < 0 || n >= behind) {
            if (b < 0) b = find_row(f.starts, (int)a.B, n);
            else while (f.starts[b + 1] <= n) b++;
            start = f.starts[b]; behind = f.starts[b + 1];
            taken = f.taken[b];
            held = f.held ? f.held[b] : max(a.lengths_out[b], 0) - (taken >= 0 ? max(a.new_tokens[b], 0) : 0);
            owned = pages_of(held, p.page);
        }
        position[k] = held + n - start;
        if (taken >= 0) {
            const int at = kvc_divide(position[k], p.page), row = position[k] - at * (int)a.page_size;
            int32_t *const entry = a.table + b * a.table_stride + at;
            const int page = at >= owned ? a.free_pages[taken + at - owned] : *entry;
            if (at >= owned && row == 0) *entry = page;     // (a new page begins with one of these tokens)
            if ((unsigned)page < (unsigned)a.n_pages) slot[k] = page * (int)a.page_size + row;
            else flags = KVC_FLAG_BAD_PAGE;
        }
    }
    if (first + 4 <= a.tokens && ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0) {
        *reinterpret_cast<int4 *>(a.slots + first) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<int4 *>(a.positions + first) = make_int4(position[0], position[1], position[2], position[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (first + k < a.tokens) { a.slots[first + k] = slot[k]; a.positions[first + k] = position[k]; }
    }
    raise_flag(a.status, flags);
}

template <int THREADS, bool ALONE>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(const __grid_constant__ PlanParams p) {
    __shared__ longlong2 warps[32];
    __shared__ long long largest[32];
    __shared__ int32_t starts_s[ALONE ? THREADS + 1 : 1], taken_s[ALONE ? THREADS : 1], held_s[ALONE ? THREADS : 1];
    const kvc_page_plan_args &a = p.a;
    const bool near = ALONE && a.B <= THREADS;              // (what it has just written to memory comes back from L2, trip by trip: 16 requests 4.4 us, so 3.8)
    kvc_behind();
    const int B = (int)a.B;
    const long long head = min(max((long long)a.head[0], 0ll), (long long)a.n_pages);
    long long rows = 0, pages = 0, given = 0;               // in front of these 1024 requests; what this thread's have been given, with all before them
    int flags = a.head[0] != head ? KVC_FLAG_BAD_LENGTH : 0;
    for (int b0 = 0; b0 < B; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        int held = 0, add = 0;
        if (b < B) { held = a.lengths[b]; add = a.new_tokens[b]; }
        if (held < 0 || add < 0) flags |= KVC_FLAG_BAD_LENGTH;
        held = max(held, 0); add = max(add, 0);
        const bool counted = (long long)held + add < (1ll << 31);
        const int owned = pages_of(held, p.page), wanted = counted ? pages_of(held + add, p.page) : 0;
        bool fits = counted && wanted <= a.table_width;
        const long long need = fits ? wanted - owned : 0;
        long long start = add, before = need, total_rows, total_pages;
        block_scan2(start, before, total_rows, total_pages, warps);
        start += rows; before += pages;
        fits = fits && start + add <= a.tokens;             // (the requests behind the first whose rows do not fit are refused too: that their needs were summed makes no difference)
        const bool served = fits && (need == 0 || head + before + need <= a.n_pages);
        if (b < B) {
            a.starts[b] = (int32_t)min(start, (long long)a.tokens);
            a.taken[b] = served ? (int32_t)min(head + before, (long long)a.n_pages) : -1;
            a.lengths_out[b] = served ? held + add : held;
            if (near) { starts_s[b] = (int32_t)min(start, (long long)a.tokens); taken_s[b] = served ? (int32_t)min(head + before, (long long)a.n_pages) : -1; held_s[b] = held; }
            if (!served) flags |= KVC_FLAG_NO_PAGES;
        }
        if (served && need > 0) given = before + need;
        rows += total_rows; pages += total_pages;
    }
    // those that were given pages are the first of those that asked for some: what was taken is the largest sum
    given = block_max(given, largest);
    if (threadIdx.x == 0) {
        a.starts[B] = (int32_t)min(rows, (long long)a.tokens);
        if (near) starts_s[B] = (int32_t)min(rows, (long long)a.tokens);
        a.head_out[0] = (int32_t)(head + given);
    }
    raise_flag(a.status, flags);
    if (ALONE) {
        __syncthreads();
        const int end = (int)min(rows, (long long)a.tokens);
        const Found f = {near ? starts_s : a.starts, near ? taken_s : a.taken, near ? held_s : nullptr};
        for (int n = threadIdx.x * 4; n < (int)a.tokens; n += THREADS * 4) plan_rows(p, f, n, end);
    }
}

__global__ void __launch_bounds__(FILL_THREADS) plan_rows_kernel(const __grid_constant__ PlanParams p) {
    kvc_behind();
    const long long n = 4 * ((long long)blockIdx.x * FILL_THREADS + threadIdx.x);
    if (n < p.a.tokens) plan_rows(p, {p.a.starts, p.a.taken, nullptr}, (int)n, p.a.starts[p.a.B]);
}

struct ReleaseParams { kvc_page_release_args a; kvc_div page; };

// entries [i, i + 4) of the `freed` pages that go back; `to` is where the first one goes
__device__ __forceinline__ void release_rows(const ReleaseParams &p, int i, int freed, int32_t *to) {
    const kvc_page_release_args &a = p.a;
    int b = find_row(a.first, (int)a.B, i);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (i + k >= freed) return;
        while (a.first[b + 1] <= i + k) b++;
        to[i + k] = a.table[b * a.table_stride + i + k - a.first[b]];
    }
}

template <int THREADS, bool ALONE>
__global__ void __launch_bounds__(THREADS) page_release_kernel(const __grid_constant__ ReleaseParams p) {
    __shared__ longlong2 warps[32];
    __shared__ long long largest[32];
    const kvc_page_release_args &a = p.a;
    kvc_behind();
    const int B = (int)a.B;
    const long long head = min(max((long long)a.head[0], 0ll), (long long)a.n_pages);
    long long pages = 0, freed = 0;
    int flags = a.head[0] != head ? KVC_FLAG_BAD_LENGTH : 0;
    for (int b0 = 0; b0 < B; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        const bool done = b < B && a.done[b] != 0;
        int held = b < B ? a.lengths[b] : 0;
        if (held < 0) { flags |= KVC_FLAG_BAD_LENGTH; held = 0; }
        long long back = done ? pages_of(held, p.page) : 0;
        if (back > a.table_width) { flags |= KVC_FLAG_BAD_LENGTH; back = a.table_width; }
        long long before = back, zero = 0, total, unused;
        block_scan2(before, zero, total, unused, warps);
        before += pages;
        const bool fits = before + back <= head;
        if (done && !fits) flags |= KVC_FLAG_NO_PAGES;
        if (b < B) {
            a.first[b] = (int32_t)min(before, head);
            a.lengths_out[b] = done && fits ? 0 : held;
        }
        if (fits) freed = before + back;
        pages += total;
    }
    freed = block_max(freed, largest);
    if (threadIdx.x == 0) {
        a.first[B] = (int32_t)freed;
        a.head_out[0] = (int32_t)(head - freed);
    }
    raise_flag(a.status, flags);
    if (ALONE) {
        __syncthreads();
        for (int i = threadIdx.x * 4; i < (int)freed; i += THREADS * 4) release_rows(p, i, (int)freed, a.free_pages + (head - freed));
    }
}

__global__ void __launch_bounds__(FILL_THREADS) release_rows_kernel(const __grid_constant__ ReleaseParams p) {
    kvc_behind();
    const int freed = p.a.first[p.a.B];
    for (long long i = 4 * ((long long)blockIdx.x * FILL_THREADS + threadIdx.x); i < freed; i += 4ll * gridDim.x * FILL_THREADS)
        release_rows(p, (int)i, freed, p.a.free_pages + p.a.head_out[0]);
}

// ---- rotation ---------------------------------------------------------------------------------------------------
//
// Every value is read once and written once: HBM for a prompt, latency for a step.  cos and sin are made once for a token and several of its
// heads, in registers, while the first of these are on their way.

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
__device__ __forceinline__ float2 turn(double position, double turns, float factor) {
    double whole = position * turns;
    whole -= rint(whole);
    const float t = (float)whole, quarter = rintf(4.0f * t), x = fmaf(-0.25f, quarter, t) * 6.2831853071795865f, y = x * x;
    const int q = (int)quarter;
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

// Queries, keys or values: a CTA has rows of one of them.  dst: token stride 0 for the pools, where `places` say where a token goes.
struct Part {
    const void *src;
    void *dst;
    int64_t src_token, src_head, dst_token, dst_head;
    int heads, chunk, of_token, turned;                     // heads, those that a thread takes, threads' shares of a token, rotated units of a head
    unsigned first;                                         // CTA
    kvc_div chunks;                                         // by of_token
};

struct RotaryParams {
    kvc_rotary_args a;
    kvc_div page, units;                                    // divisors: page size, D / 16
    long long slots;                                        // of the pool
    Part parts[3];
};

// Where a token goes: element offsets of its row in the pools, -1: nowhere
struct Place { long long k, v; };

__device__ __forceinline__ Place place_of(const RotaryParams &p, long long n, int &flags) {
    const kvc_rotary_args &a = p.a;
    Place r = {-1, -1};
    const int slot = a.slots[n];
    if (slot < 0) return r;
    if (slot >= p.slots) { flags = KVC_FLAG_BAD_PAGE; return r; }
    const int page = kvc_divide(slot, p.page), row = slot - page * (int)a.page_size;
    r.k = page * a.kp_page + row * a.kp_row;
    r.v = page * a.vp_page + row * a.vp_row;
    return r;
}

constexpr int ROTARY_THREADS = 256, ROTARY_CTAS = 3, CHUNK = 4;

// Heads of 16 n channels, rotated by multiples of 16, everything on 16 bytes.  A thread has a unit of 16 channels (8 pairs: two pieces of 16
// bytes, half the rotated channels apart, or next to each other) of up to CHUNK heads of a token: its 8 angles serve them all, and no thread waits for another.
// Queries, keys and values have CTAs of their own, so that all that is picked by kind is picked for a CTA.
// Measured: 16384 tokens of 40 + 10 + 10 heads of 128 channels (503 MB) 78.5 us, 6.4 TB/s; with the angles of a CTA's tokens in shared memory, made behind a
// barrier, 84.5 to 89; CHUNK 8 79.2, 5 82.7; at most two heads under way 79.5, two CTAs per SM 88, four (spilling) 97.  32749 tokens of 8 heads (134 MB) 22.7 us, before 28.6.
template <typename T>
__global__ void __launch_bounds__(ROTARY_THREADS, ROTARY_CTAS) rotary_rows_kernel(const __grid_constant__ RotaryParams p) {
    kvc_behind();
    const kvc_rotary_args &a = p.a;
    const int which = blockIdx.x >= p.parts[2].first ? 2 : (blockIdx.x >= p.parts[1].first ? 1 : 0);
    const Part &part = p.parts[which];
    const int units = (int)a.D / 16, turned = part.turned, id = (int)((blockIdx.x - part.first) * ROTARY_THREADS + threadIdx.x);
    const int group = kvc_divide(id, p.units), u = id - group * units, n = kvc_divide(group, part.chunks);
    if (n >= a.N) return;
    const int h0 = (group - n * part.of_token) * part.chunk, heads = min(part.chunk, part.heads - h0);
    const bool half = a.layout == KVC_ROTARY_HALF && u < turned;
    const int c0 = half ? 8 * u : 16 * u, apart = half ? 8 * turned : 8;
    const T *src = reinterpret_cast<const T *>(part.src) + n * part.src_token + h0 * part.src_head + c0;
    T *dst = reinterpret_cast<T *>(part.dst) + n * part.dst_token + h0 * part.dst_head + c0;
    uint4 x[CHUNK][2];
#pragma unroll
    for (int j = 0; j < CHUNK; j++) {
        if (j < heads) {
            x[j][0] = *reinterpret_cast<const uint4 *>(src);
            x[j][1] = *reinterpret_cast<const uint4 *>(src + apart);
        }
        src += part.src_head;
    }
    if (which > 0) {
        int flags = 0;
        const Place at = place_of(p, n, flags);
        raise_flag(a.status, flags);
        if (at.k < 0) return;
        dst += which == 1 ? at.k : at.v;
    }
    const bool turns = u < turned;
    float2 cs[8];
    if (turns) {
        const double position = a.inverse ? -(double)a.positions[n] : (double)a.positions[n];
#pragma unroll
        for (int k = 0; k < 8; k++) cs[k] = turn(position, a.frequencies[8 * u + k] * TURNS_OF_RADIANS, a.factor);
    }
#pragma unroll
    for (int j = 0; j < CHUNK; j++) {
        if (j < heads) {
            uint32_t w[8] = {x[j][0].x, x[j][0].y, x[j][0].z, x[j][0].w, x[j][1].x, x[j][1].y, x[j][1].z, x[j][1].w};
            if (turns) {
                // pairs: with halves a value of the first piece and its like of the second, else neighbours
                if (half) {
#pragma unroll
                    for (int m = 0; m < 4; m++) {
                        const float2 f = unpack(w[m], T()), g = unpack(w[4 + m], T()), c = cs[2 * m], d = cs[2 * m + 1];
                        w[m] = pack(f.x * c.x - g.x * c.y, f.y * d.x - g.y * d.y, T());
                        w[4 + m] = pack(g.x * c.x + f.x * c.y, g.y * d.x + f.y * d.y, T());
                    }
                } else {
#pragma unroll
                    for (int m = 0; m < 8; m++) {
                        const float2 f = unpack(w[m], T());
                        w[m] = pack(f.x * cs[m].x - f.y * cs[m].y, f.y * cs[m].x + f.x * cs[m].y, T());
                    }
                }
            }
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4 *>(dst + apart) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        dst += part.dst_head;
    }
}

// Any sizes and strides: a thread per pair or copied channel.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const __grid_constant__ RotaryParams p) {
    kvc_behind();
    const kvc_rotary_args &a = p.a;
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
        int flags = 0;
        const Place at = place_of(p, n, flags);
        raise_flag(a.status, flags);
        if (at.k < 0) return;
        x = key ? reinterpret_cast<const T *>(a.k) + n * a.k_token + hk * a.k_head : reinterpret_cast<const T *>(a.v) + n * a.v_token + hk * a.v_head;
        y = key ? reinterpret_cast<T *>(a.kpages) + at.k + hk * a.kp_head : reinterpret_cast<T *>(a.vpages) + at.v + hk * a.vp_head;
    }
    if (u >= half) { y[half + u] = x[half + u]; return; }
    const int i0 = a.layout == KVC_ROTARY_HALF ? u : 2 * u, i1 = a.layout == KVC_ROTARY_HALF ? u + half : 2 * u + 1;
    const T x0 = x[i0], x1 = x[i1];
    if (h >= a.Hq + a.Hkv) { y[i0] = x0; y[i1] = x1; return; }
    const float2 cs = turn(a.inverse ? -(double)a.positions[n] : (double)a.positions[n], a.frequencies[u] * TURNS_OF_RADIANS, a.factor);
    const float f0 = to_float(x0), f1 = to_float(x1);
    y[i0] = from_float<T>(f0 * cs.x - f1 * cs.y);
    y[i1] = from_float<T>(f1 * cs.x + f0 * cs.y);
}

}  // namespace

extern "C" int kvc_page_plan(const kvc_page_plan_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_page_plan: null pointer");
    PlanParams p;
    memcpy(&p.a, args, sizeof(p.a));
    const kvc_page_plan_args &a = p.a;
    KVC_REQUIRE(a.B >= 0 && a.B < (1 << 24) && a.n_pages >= 0 && a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.tokens >= 0 && a.tokens < (1ll << 31) - 4,
                "kvc_page_plan: bad sizes");
    KVC_REQUIRE(a.n_pages * a.page_size < (1ll << 31), "kvc_page_plan: slots have 32 bits, the pool %lld tokens", (long long)(a.n_pages * a.page_size));
    KVC_REQUIRE(a.table_width >= 0 && a.table_width < (1ll << 31) && (a.B <= 1 || a.table_stride >= a.table_width), "kvc_page_plan: rows of the table overlap");
    KVC_REQUIRE(a.head && a.head_out && a.starts && (a.B == 0 || (a.lengths && a.new_tokens && a.lengths_out && a.taken)) && (a.free_pages || a.n_pages == 0) &&
                    (a.table || a.B == 0 || a.table_width == 0) && (a.tokens == 0 || (a.slots && a.positions)), "kvc_page_plan: null pointer");
    p.page = kvc_make_div((uint32_t)a.page_size);
    cudaStream_t s = kvc_cu(stream);
    if (a.tokens > FILL_ALONE) {
        if (int rc = kvc_launch_early(page_plan_kernel<SCAN_THREADS, false>, 1, SCAN_THREADS, s, p)) return rc;
        return kvc_launch_early(plan_rows_kernel, (unsigned)((a.tokens + 4 * FILL_THREADS - 1) / (4 * FILL_THREADS)), FILL_THREADS, s, p);
    }
    if (a.B <= SMALL_THREADS && a.tokens <= 4 * SMALL_THREADS) return kvc_launch_early(page_plan_kernel<SMALL_THREADS, true>, 1, SMALL_THREADS, s, p);
    return kvc_launch_early(page_plan_kernel<SCAN_THREADS, true>, 1, SCAN_THREADS, s, p);
}

extern "C" int kvc_page_release(const kvc_page_release_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_page_release: null pointer");
    ReleaseParams p;
    memcpy(&p.a, args, sizeof(p.a));
    const kvc_page_release_args &a = p.a;
    KVC_REQUIRE(a.B >= 0 && a.B < (1 << 24) && a.n_pages >= 0 && a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages * a.page_size < (1ll << 31),
                "kvc_page_release: bad sizes");
    KVC_REQUIRE(a.table_width >= 0 && a.table_width < (1ll << 31) && (a.B <= 1 || a.table_stride >= a.table_width), "kvc_page_release: rows of the table overlap");
    KVC_REQUIRE(a.head && a.head_out && a.first && (a.B == 0 || (a.lengths && a.done && a.lengths_out)) && (a.free_pages || a.n_pages == 0) &&
                    (a.table || a.B == 0 || a.table_width == 0), "kvc_page_release: null pointer");
    p.page = kvc_make_div((uint32_t)a.page_size);
    cudaStream_t s = kvc_cu(stream);
    // (how many pages come back is known on the device only: at most so many)
    const int64_t most = a.table_width == 0 ? 0 : std::min(a.n_pages, a.B * a.table_width);
    if (most > FILL_ALONE) {
        if (int rc = kvc_launch_early(page_release_kernel<SCAN_THREADS, false>, 1, SCAN_THREADS, s, p)) return rc;
        return kvc_launch_early(release_rows_kernel, (unsigned)std::min<int64_t>((most + 4 * FILL_THREADS - 1) / (4 * FILL_THREADS), 4ll * kvc_sm_count()), FILL_THREADS, s, p);
    }
    if (a.B <= SMALL_THREADS && most <= 8 * SMALL_THREADS) return kvc_launch_early(page_release_kernel<SMALL_THREADS, true>, 1, SMALL_THREADS, s, p);
    return kvc_launch_early(page_release_kernel<SCAN_THREADS, true>, 1, SCAN_THREADS, s, p);
}

extern "C" int kvc_rotary_store(const kvc_rotary_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_rotary_store: null pointer");
    RotaryParams p;
    memcpy(&p.a, args, sizeof(p.a));
    kvc_rotary_args &a = p.a;
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_rotary_store: unknown type %d", a.type);
    KVC_REQUIRE(a.layout == KVC_ROTARY_HALF || a.layout == KVC_ROTARY_INTERLEAVED, "kvc_rotary_store: unknown layout %d", a.layout);
    KVC_REQUIRE(a.N >= 0 && a.Hq >= 0 && a.Hkv >= 0 && a.D > 0 && a.D <= 65536 && a.rotary >= 0 && a.rotary <= a.D && a.rotary % 2 == 0,
                "kvc_rotary_store: bad sizes (head of %lld channels, %lld rotated)", (long long)a.D, (long long)a.rotary);
    KVC_REQUIRE(a.Hkv == 0 || (a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages >= 0 && a.n_pages * a.page_size < (1ll << 31)), "kvc_rotary_store: bad pool");
    if (a.N == 0 || a.Hq + a.Hkv == 0) return KVC_OK;
    KVC_REQUIRE((a.Hq == 0 || (a.q && a.q_out)) && (a.Hkv == 0 || (a.k && a.v && a.slots && ((a.kpages && a.vpages) || a.n_pages == 0))) &&
                    (a.rotary == 0 || (a.positions && a.frequencies)), "kvc_rotary_store: null pointer");
    KVC_REQUIRE(a.Hq < (1 << 20) && a.Hkv < (1 << 20) && a.N < (1ll << 31), "kvc_rotary_store: too many heads or tokens");
    const long long H = a.Hq + 2 * a.Hkv, rows = a.N * H;
    p.page = kvc_make_div((uint32_t)std::max<int64_t>(a.page_size, 1));
    p.slots = a.n_pages * a.page_size;
    // (the stride of a dimension of one, and what a part that is not there says, may be anything)
    if (a.Hq == 0) a.q = nullptr, a.q_out = nullptr;
    if (a.Hkv == 0) a.k = a.v = nullptr, a.kpages = a.vpages = nullptr;
    if (a.Hq <= 1) a.q_head = a.out_head = 0;
    if (a.N == 1 || a.Hq == 0) a.q_token = a.out_token = 0;
    if (a.Hkv <= 1) a.k_head = a.v_head = a.kp_head = a.vp_head = 0;
    if (a.N == 1 || a.Hkv == 0) a.k_token = a.v_token = 0;
    if (a.page_size <= 1 || a.Hkv == 0) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1 || a.Hkv == 0) a.kp_page = a.vp_page = 0;
    // What is written in no order must not overlap: rows of the results or of a pool each other, a result what another thread reads.
    const kvc_rows q = kvc_make_rows(a.q, a.D, a.N, a.q_token, a.Hq, a.q_head), out = kvc_make_rows(a.q_out, a.D, a.N, a.out_token, a.Hq, a.out_head);
    const kvc_rows k = kvc_make_rows(a.k, a.D, a.N, a.k_token, a.Hkv, a.k_head), v = kvc_make_rows(a.v, a.D, a.N, a.v_token, a.Hkv, a.v_head);
    const kvc_rows kp = kvc_make_rows(a.kpages, a.D, a.n_pages, a.kp_page, a.page_size, a.kp_row, a.Hkv, a.kp_head);
    const kvc_rows vp = kvc_make_rows(a.vpages, a.D, a.n_pages, a.vp_page, a.page_size, a.vp_row, a.Hkv, a.vp_head);
    KVC_REQUIRE(a.Hq == 0 || out.apart, "kvc_rotary_store: rows of the output overlap");
    KVC_REQUIRE(a.Hq == 0 || kvc_rows_equal(q, out) || !kvc_rows_overlap(q, out), "kvc_rotary_store: the output overlaps the queries and is not them");
    KVC_REQUIRE(a.Hq == 0 || a.Hkv == 0 || !(kvc_rows_overlap(k, out) || kvc_rows_overlap(v, out)), "kvc_rotary_store: the output overlaps the keys or the values");
    KVC_REQUIRE(a.Hkv == 0 || (kp.apart && vp.apart), "kvc_rotary_store: rows of a pool overlap");
    KVC_REQUIRE(a.Hkv == 0 || !kvc_rows_overlap(kp, vp) || (a.rotary == 0 && kvc_rows_equal(kp, vp) && kvc_rows_equal(k, v)), "kvc_rotary_store: the pools overlap");
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages);
    const int64_t strides = a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head | a.out_token | a.out_head | a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head;
    cudaStream_t s = kvc_cu(stream);
    if ((at & 15) == 0 && (strides & 7) == 0 && a.D % 16 == 0 && a.rotary % 16 == 0 && rows * (a.D / 16) < (1ll << 31) - ROTARY_THREADS) {
        const int units = (int)a.D / 16;
        p.units = kvc_make_div((uint32_t)units);
        p.parts[0] = {a.q, a.q_out, a.q_token, a.q_head, a.out_token, a.out_head, (int)a.Hq};
        p.parts[1] = {a.k, a.kpages, a.k_token, a.k_head, 0, a.kp_head, (int)a.Hkv};
        p.parts[2] = {a.v, a.vpages, a.v_token, a.v_head, 0, a.vp_head, (int)a.Hkv};
        // heads of a thread: CHUNK share its angles, unless that leaves too few threads for the device's latency
        const long long threads = (long long)ROTARY_CTAS * ROTARY_THREADS * kvc_sm_count();
        const int chunk = (int)std::max<long long>(1, std::min<long long>(CHUNK, rows * units / threads));
        int64_t grid = 0;
        for (int i = 0; i < 3; i++) {
            Part &part = p.parts[i];
            const int chunks = std::max((part.heads + chunk - 1) / chunk, 1);
            part.chunk = std::max((part.heads + chunks - 1) / chunks, 1);
            part.of_token = chunks;
            part.chunks = kvc_make_div((uint32_t)chunks);
            part.turned = i < 2 ? (int)a.rotary / 16 : 0;
            part.first = (unsigned)grid;
            if (part.heads > 0) grid += (a.N * chunks * units + ROTARY_THREADS - 1) / ROTARY_THREADS;
        }
        return kvc_launch_early(a.type == KVC_TYPE_FP16 ? rotary_rows_kernel<__half> : rotary_rows_kernel<__nv_bfloat16>, (unsigned)grid, ROTARY_THREADS, s, p);
    }
    const long long n = rows * (a.D - a.rotary / 2);
    KVC_REQUIRE((n + 255) / 256 < (1ll << 31), "kvc_rotary_store: too many elements");
    return kvc_launch_early(a.type == KVC_TYPE_FP16 ? rotary_any_kernel<__half> : rotary_any_kernel<__nv_bfloat16>, (unsigned)((n + 255) / 256), 256, s, p);
}
