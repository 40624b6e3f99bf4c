// Attention of one new token per request over a paged key-value cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m) with s_t = scaling * q . k_t: one pass over the tokens with a running maximum m
// and a running sum l; whenever the maximum grows, sum and accumulators are multiplied with exp(m_old - m_new).
//
// What bounds it: every key and value is read once and used for Hq / Hkv heads, 4 (Hq / Hkv) operations per 4 bytes: HBM, for any
// number of heads that a model has.  Everything else is arranged so that the loads never pause:
//
// Work is cut into tiles of 64 tokens of a column (a request's KV head; or 32 tokens of two heads, see choose_heads), all tiles of all columns in one row; each CTA takes
// an equal, contiguous share of the row, found from the lengths in the kernel (the host does not know them).  Lengths may be as unequal as they like, and a
// single long request is spread over the device.  A column that lies in one share is written at once; one that was cut leaves partial results {m, l,
// sums} in the workspace, and the CTA that finishes last (a counter, put back to zero) joins them in the order of the shares, so that
// the result does not depend on who that was.
//
// Four warps take 16 of a tile's tokens each, with a ring of stages of their own that they fill with 16-byte asynchronous copies (any strides,
// pages that end anywhere) and drain without a barrier; the copies go on over the ends of columns.  The
// block table's entries are asked for a tile ahead of the copies that need them.
//
// The products: 16 tokens x 8 heads, mma.m16n8k16 with the keys as the operand with 16 rows, and O^T = V^T P^T with 16 channels x 8
// heads, so that few heads waste little.  (tcgen05 wants 64 rows and its operands in shared memory behind barriers of the whole CTA; here the tensor
// work is a few per cent of the time that the bytes need.)  P is split into two 16-bit pieces, hi + lo, and multiplied twice: the weights keep 21
// (fp16) or 16 bits (bf16), and the result is rounded once, at the end.  fp16 weights are carried times 2^14, so that the pieces of weights down to 2^-28
// of the largest are normal numbers and many small ones are not lost.  Two pieces make no number of an infinite value (0 times it, or pieces of two signs), and neither does a
// weight that is nothing in 32 bits: a column whose sums are no numbers although its weights are is looked at again (infinite_values).
#pragma once

#include <math_constants.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "kvc_paged.cuh"

namespace kvc_paged {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int MAX_CTAS_PER_SM = 4;
constexpr int DRAWN_REQUESTS = 512;             // of more requests nothing is drawn: where a tile belongs is looked up in shared memory
// Tiles of a share from which on the last eighth is drawn.  148 tiles (16 x 32768 tokens of 8 KV heads): 317 us, 333 undrawn; 64 (64 requests of up to 4096 tokens,
// 10 KV heads): 157 and 148, 37 (8 x 4096 of 32): 89.3 and 89.6.
constexpr int DRAWN_SHARE = 96;
constexpr int JOINED = 8;                       // partial results that are asked for at once
// Tiles of a share at least: a tile more takes less than joining two parts (8 heads of 100 tokens 5.6 us, with 1 7.5, with 4, of 777 tokens of 32 heads, 12.2 for 10.9).
constexpr int MIN_TILES = 2;
constexpr int MAX_GROUP = 16;                   // query heads that a column serves (of all its KV heads)

struct Params {
    kvc_paged_attn_args a;
    kvc_div page;
    int chunk;                                  // requests of a lane
    int group, columns, per_head;               // query heads of a column at most, columns of a request, columns of a KV head
    int most_tokens;                            // of a table row
    unsigned n_pages;
    int negative;                               // scaling: the scores' maximum is taken before they are scaled
    float log2_scaling, per_cta;                // per_cta: a little less than one over the number of CTAs
    long long v_less_k;                         // bytes from the keys' pool to the values'
    const int32_t *starts;                      // the requests' first rows of q and out; null (a kernel without ROWS): row b is request b's
    int rows;                                   // of q and out
    int *drawn;                                 // how many pieces have been drawn
    unsigned *counters, *group_counters;        // of the places of partial results
    int part;                                   // floats of a place: sums of values, maxima and sums of weights
    float *parts;
    kvc_scales s;                               // of pools of codes
    float *wide;                                // WIDE_RESULTS: [request][query head][D], as the logarithms are by request then
};

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static constexpr float LIFT = 14.0f;
    static constexpr uint32_t INFINITE = 0x7c00;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 r = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&r); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Pair<__nv_bfloat16> {
    static constexpr float LIFT = 0.0f;
    static constexpr uint32_t INFINITE = 0x7f80;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 r = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&r); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// 16 bytes to shared memory, zeros when `on` is false (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// where a 16-byte piece of a row of ROW bytes lies in a stage: the 8 rows of a matrix load fall on different banks
template <int ROW> __device__ __forceinline__ uint32_t piece_at(int row, int piece) {
    if constexpr (ROW % 128 == 0) return (uint32_t)(row * (ROW / 16) + (piece ^ (row & 7))) * 16;     // rows start on bank 0
    else if constexpr (ROW % 64 == 0) return (uint32_t)(row * (ROW / 16) + (piece ^ ((row >> 1) & 3))) * 16;      // every other row starts in the middle
    else return (uint32_t)(row * (ROW / 16) + (piece ^ ((row >> 2) & 1))) * 16;                     // 96: a quarter on, from row to row
}

// ---- rows of codes
// Codes are numbers of 16 bits (int8 whole ones, e4m3 with four bits), so the products are the same and exact: fp16 whatever the queries' type.  Four codes of a register become two
// pairs, neighbours for keys, and every other one for values (what lies next to each other there are two channels of a token, and a pair is of two tokens).
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(on ? 4 : 0) : "memory");
}
// bytes FIRST and FIRST + STEP of a register
template <int KIND, int FIRST, int STEP> __device__ __forceinline__ uint32_t two_codes(uint32_t c) {
    if constexpr (KIND == KVC_CODES_INT8) {                  // (c: codes + 128) a byte as the last bits of 1024
        const uint32_t v = __byte_perm(c, 0x64646464u, 0x4040 + FIRST + ((FIRST + STEP) << 8));
        const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), __float2half2_rn(1152.0f));
        return *reinterpret_cast<const uint32_t *>(&r);
    } else {
        uint32_t r;                                         // (c: as asked for, each pair in a half)
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, " "l; }" : "=r"(r) : "r"((STEP == 1 ? FIRST : 2 * FIRST) == 0 ? c : c >> 16));
        return r;
    }
}
// the power of two that brings x to [2^14, 2^15), or a smaller one where there is none, and one over it
__device__ __forceinline__ uint32_t exponent_of(float x) { return min(max(__float_as_uint(x) >> 23, 15u), 254u); }
__device__ __forceinline__ float lifted(float x) { return __uint_as_float((268 - exponent_of(x)) << 23); }
__device__ __forceinline__ float lifted_back(float x) { return __uint_as_float((exponent_of(x) - 14) << 23); }
// a register of codes as two_codes of that STEP wants it
template <int KIND, int STEP> __device__ __forceinline__ uint32_t offset_codes(uint32_t c) {
    if constexpr (KIND == KVC_CODES_INT8) return c ^ 0x80808080u;
    return STEP == 1 ? c : __byte_perm(c, 0, 0x3120);
}

// The first of a request's rows of q and out, for b = B the first that is nobody's.  (Kept inside the tensors whatever `starts` hold, as lengths are.)
template <bool ROWS> __device__ __forceinline__ int row_of(const Params &p, int b) { return ROWS && p.starts ? min(max(p.starts[b], 0), p.rows) : b; }

// The tokens of a request that count: [first, len).  None where it has no row, or more than one.
struct Span { int first, len; };
template <bool ROWS> __device__ __forceinline__ Span span_of(const Params &p, int b, int &flags) {
    int len = p.a.lengths[b];
    if (len < 0 || len > p.most_tokens) { flags |= KVC_FLAG_BAD_LENGTH; len = len < 0 ? 0 : p.most_tokens; }
    if (ROWS) {
        const int rows = row_of<ROWS>(p, b + 1) - row_of<ROWS>(p, b);
        if (rows > 1) flags |= KVC_FLAG_BAD_LENGTH;
        if (rows != 1) len = 0;
    }
    Span s;
    s.len = len;
    s.first = p.a.window > 0 && len > p.a.window ? len - (int)p.a.window : 0;
    return s;
}
template <int TILE> __device__ __forceinline__ int tiles_of(const Span &s) { return (s.len - s.first + TILE - 1) / TILE; }

// n / d of numbers that are not negative, through a float that some steps put right (16 of them: it is off by 3 2^-24, and quotients are below 2^26).  Lengths are read more
// than once and must not change while the kernel runs: its warps would take different numbers of turns between the CTA's barriers.
__device__ __forceinline__ int quotient(int n, int d) {
    if (d <= 0) return 0;
    int q = (int)((float)n * __frcp_rn((float)d));
    for (int k = 0; k < 16 && (unsigned)q * (unsigned)d > (unsigned)n; k++) q--;
    for (int k = 0; k < 16 && (unsigned)n - (unsigned)q * (unsigned)d >= (unsigned)d; k++) q++;
    return q;
}

// A place in the row of tiles: tile `i` of column `c` of request `b`
struct Place { int b, c, i, n; Span span; };
template <int TILE, bool ROWS> __device__ __forceinline__ void next_tile(const Params &p, Place &at) {
    if (++at.i < at.n) return;
    at.i = 0;
    if (++at.c < p.columns) return;
    at.c = 0;
    int unused = 0;
    at.n = 0;
    while (++at.b < (int)p.a.B) {
        at.span = span_of<ROWS>(p, at.b, unused);
        if ((at.n = tiles_of<TILE>(at.span)) > 0) return;
    }
    at.b = (int)p.a.B - 1;                                  // (behind the last: a place without tokens)
    at.span = {0, 0};
}

// The channels of query heads [h0, h0 + heads) of request b that came out as no numbers although their weights are some (`odd`: a bit for each such head), by the definition:
// a value of +inf or -inf that counts makes the sum that, both, or one that is no number itself, or one of weight 0 (a score of -inf), none.  The CTA reads the column's values
// again, of the 16-byte pieces that hold such a channel, eight at a time a thread; `seen` (heads * D bytes of shared memory and a word) has for each channel 1: +inf, 2: -inf.  All
// threads call it, behind a barrier.  (One infinity among 131072 tokens of 8 KV heads: a call of 90 us takes 1200; 8 x 4096 of 32
// heads, one for each, 87 and 123; values that are all no numbers 140 and 133.)
template <typename T, int D, bool ROWS>
__device__ __noinline__ void infinite_values(const Params &p, int b, int row, int h0, int heads, unsigned odd, uint32_t *seen) {
    constexpr uint32_t INFINITE = Pair<T>::INFINITE;
    const kvc_paged_attn_args &a = p.a;
    const int tid = threadIdx.x, g = (int)(a.Hq / a.Hkv), hk0 = h0 / g;
    uint32_t *const pieces_s = seen + heads * (D / 4);      // a bit for each piece of the KV heads' rows (32 at most)
    auto result = [&](int i) { return reinterpret_cast<uint16_t *>(reinterpret_cast<T *>(a.out) + row * a.out_token + (h0 + i / D) * a.out_head + i % D); };
    auto no_number = [&](int i) { return (odd >> i / D & 1) && (*result(i) & 0x7fff) > INFINITE; };
    for (int i = tid; i <= heads * (D / 4); i += THREADS) seen[i] = 0;
    __syncthreads();
    for (int i = tid; i < heads * D; i += THREADS)
        if (no_number(i)) atomicOr(pieces_s, 1u << (((h0 + i / D) / g - hk0) * (D / 8) + i % D / 8));
    __syncthreads();
    const unsigned pieces = *pieces_s;
    if (pieces == 0) return;                                // (infinities of two signs in one thread's channels)
    const int many = max(__popc(pieces), 1), ways = THREADS / many, way = tid / many;
    int piece = 0;
    for (int left = tid % many; piece < 31 && !((pieces >> piece & 1) && left-- == 0); piece++) {}
    const int hk = hk0 + piece / (D / 8), channel = piece % (D / 8) * 8, from = max(h0, hk * g), to = min(h0 + heads, (hk + 1) * g);
    int unused = 0;
    const Span span = span_of<ROWS>(p, b, unused);
    auto page_of = [&](int t) { return a.table[b * a.table_stride + kvc_divide(t, p.page)]; };
    auto row_at = [&](const void *pool, long long of_page, long long of_row, long long of_head, int page, int t) {
        return reinterpret_cast<const T *>(pool) + page * of_page + (t - kvc_divide(t, p.page) * (int)a.page_size) * of_row + hk * of_head;
    };
    auto odd_pair = [](uint32_t v) { return (v & INFINITE) == INFINITE || (v >> 16 & INFINITE) == INFINITE; };
    auto odd_piece = [&](const uint4 &v) { return odd_pair(v.x) || odd_pair(v.y) || odd_pair(v.z) || odd_pair(v.w); };
    uint32_t plus = 0, minus = 0;                           // this thread's channels, a bit for each; none: both
    auto keep = [&](int h, uint32_t up, uint32_t down) {
        for (int c = 0; c < 8; c++) {
            const uint32_t code = (up >> c & 1) | (down >> c & 1) << 1;
            if (code) atomicOr(seen + ((h - h0) * D + channel + c) / 4, code << c % 4 * 8);
        }
    };
#pragma unroll 1
    for (long long t0 = span.first + way; way < ways && t0 < span.len && (plus & minus) != 0xff; t0 += 8 * ways) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const long long t = t0 + k * ways;
            const int page = t < span.len ? page_of((int)t) : -1;
            v[k] = (unsigned)page < p.n_pages ? *reinterpret_cast<const uint4 *>(row_at(a.vpages, a.vp_page, a.vp_row, a.vp_head, page, (int)t) + channel) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (!odd_piece(v[k])) continue;
            const int t = (int)(t0 + k * ways);
            uint32_t up = 0, down = 0;
            for (int c = 0; c < 8; c++) {
                const uint32_t pair = c < 2 ? v[k].x : c < 4 ? v[k].y : c < 6 ? v[k].z : v[k].w, x = pair >> c % 2 * 16 & 0xffff;
                if ((x & INFINITE) != INFINITE) continue;
                const bool number = (x & 0x7fff) == INFINITE;
                up |= (!number || !(x & 0x8000)) << c;
                down |= (!number || (x & 0x8000)) << c;
            }
            plus |= up;
            minus |= down;
            const T *const key = row_at(a.kpages, a.kp_page, a.kp_row, a.kp_head, page_of(t), t);
            bool weighed = false;                           // whether the weight may be 0
            for (int c = 0; c < D / 8 && !weighed; c++) weighed = odd_piece(*reinterpret_cast<const uint4 *>(key + c * 8));
            for (int h = from; weighed && h < to; h++) {
                bool none = a.q == a.out;                   // (the result is where the query was: no number stays none)
                if (!none) {
                    const T *const q = reinterpret_cast<const T *>(a.q) + row * a.q_token + h * a.q_head;
                    float s = 0.0f;
                    for (int c = 0; c < D; c++) s = fmaf((float)q[c], (float)key[c], s);
                    none = (p.negative ? -s : s) == -CUDART_INF_F;
                }
                if (none) keep(h, up | down, up | down);
            }
        }
    }
    for (int h = from; way < ways && h < to; h++) keep(h, plus, minus);
    __syncthreads();
    for (int i = tid; i < heads * D; i += THREADS) {
        const uint32_t code = seen[i / 4] >> i % 4 * 8 & 3;
        if ((code == 1 || code == 2) && no_number(i)) *result(i) = (uint16_t)(code == 1 ? INFINITE : INFINITE | 0x8000);
    }
    __syncthreads();
}

// What a kernel's tiles are, by its channels and the kind of its rows: T, codes, or T with results of 32 bits for whoever joins them with others (a call with prefixes).
constexpr int WIDE_RESULTS = 3;
template <int D, int KIND> struct Tiles {
    static constexpr bool CODED = KIND == KVC_CODES_INT8 || KIND == KVC_CODES_E4M3;
    static constexpr int TOKENS = CODED ? 32 : 16, ROW = CODED ? D : 2 * D;                 // tokens of a warp's tile, bytes of a row
    static constexpr uint32_t HALF_STAGE = TOKENS * ROW, STAGE = 2 * HALF_STAGE + (CODED ? 8 * TOKENS : 0);     // keys, values; of codes their scales
};

// Rows of codes: a warp's tile has 32 tokens, as many bytes as 16 of 16 bits.  A token's score is its codes' times its key's scale.  Its weight is multiplied with its value's scale before
// it meets the codes, as two pieces of fp16, for which the product is too small or too large: a power of two that brings the largest product of a head so far to 2^14 is kept beside the sums as
// the maximum is, and taken out of them.  (The largest product, not the largest scale: a row of large values that a head gives no weight takes no bits of the others.)  What is 2^-39 of that
// product is lost, and a weight that is 2^-126 of the largest one.  bf16 queries become fp16 times a power of two for each head (what is 2^29 below the head's largest value loses bits, no less than a sum in 32 bits does).
// What bounds them is no longer HBM but instructions, about 1020 for a tile of 32 tokens of 128 channels, a third of them codes that become numbers: 8 x 4096 tokens of 32 heads in int8 60 us (4.6 TB/s;
// fp16 rows 85), 16 x 32768 of 8 KV heads in e4m3 213 (5.2 TB/s; 317), with other pools from call to call 220.  (By the largest scale of a warp instead of a head's largest product 2 to 4 % less.)  So CTAs have equal work sooner than with rows of 16 bits: one CTA a column of 8 x 4096 took 82 us.
template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS, bool ROWS, int KIND>
__global__ void __launch_bounds__(THREADS, CTAS) paged_attn_kernel(const __grid_constant__ Params p) {
    constexpr bool CODED = Tiles<D, KIND>::CODED;
    constexpr int KS = D / 16;                              // steps of 16 channels
    constexpr int TOKENS = Tiles<D, KIND>::TOKENS, ROW = Tiles<D, KIND>::ROW;
    constexpr int TEAM = WARPS / WH, TILE = TOKENS * TEAM;  // warps of a KV head, tokens of a tile
    constexpr uint32_t HALF_STAGE = Tiles<D, KIND>::HALF_STAGE, STAGE = Tiles<D, KIND>::STAGE, ALL = TOKENS == 32 ? 0xffffffffu : 0xffffu;
    constexpr float LIFT = CODED ? 0.0f : Pair<T>::LIFT;
    typedef std::conditional_t<CODED, uint8_t, T> Element;
    typedef std::conditional_t<CODED, Pair<__half>, Pair<T>> Operand;
    constexpr int EVEN_MOST = CODED ? 10 : D < 128 ? 10 : 14;
    static_assert(!CODED || SAME, "pools of codes have the same strides");
    static_assert(STAGES + 2 <= DRAWN_SHARE - DRAWN_SHARE / 8, "a share is long enough for the first draw");
    extern __shared__ __align__(128) uint8_t smem[];        // [warp][stage]: 16 rows of keys, 16 of values
    __shared__ uint32_t masks[WARPS][STAGES];
    __shared__ float2 ml_s[WARPS][8 * NT];                  // maximum and sum
    __shared__ float2 new_ml[MAX_GROUP];
    __shared__ Place next_start_s[WARPS];
    __shared__ unsigned before_s[CTAS >= 3 ? DRAWN_REQUESTS : 1];           // tiles of a column in front of a request
    __shared__ int last_s, next_s;
    __shared__ unsigned odd_s;                              // whether a thread has seen such a result (and which heads', while they are looked at)
    const kvc_paged_attn_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = (int)a.B;
    int flags = 0;
    if (tid == 0) odd_s = 0;                                // (the first result is written behind a barrier)

    // ---- this CTA's share
    // Whole parts of columns, one for each CTA, where parts of up to 7 / 4 of an equal share do (few columns): no CTA has two to finish then, and fewer are joined; so many
    // CTAs less still have as much under way as the memory gives (8 requests of 32 heads of 128 channels, one CTA a column: 512 tokens 15.7 us, 2048 45.6, 4096 85; in equal
    // shares 19.6, 49.4, 90).  Tiles of shorter rows are less to have under way: 5 / 4 (11 x 4096 tokens of 32 heads of 96 channels 94 us, with 7 / 4 99), and so
    // do codes; where an SM holds one CTA, 9 / 8.  Else equal shares of the row of all columns' tiles.
    // Of long shares an eighth is drawn from a counter instead, in pieces of a sixteenth of a share, then halves of it: the SMs do not get the same out of the
    // memory (of 444 CTAs with 148 tiles each the first was done at 235 us, half at 285, the last at 319).  Where columns are few all of these pieces would be
    // joined by few CTAs, and a CTA alone on its SM pauses at the end of every piece: not there.
    constexpr bool DRAWS = CTAS >= 3;
    // (All of this is on the way of the first byte.  Every warp does it by itself, for its lanes' requests: no barrier, no division but by a reciprocal.)
    int r0, r1, size;                                       // tiles [r0, r1) of the row, shares of `size`; or with even != 0: CTA r0, r1 = r0 + 1
    float even = 0.0f;                                      // one over the tiles of a part at most
    int unit = 0, least = 0, drawn_from = 0x7fffffff, all_tiles;       // tiles of the first and the last pieces that are drawn, the first tile that is not in a share
    Place at;
    auto parts_of = [&](int tiles) { return __float2int_ru((float)tiles * even); };
    {
        const int b0 = min(B, lane * p.chunk), b1 = min(B, b0 + p.chunk);
        const int n0 = b0 < b1 ? tiles_of<TILE>(span_of<ROWS>(p, b0, flags)) : 0;
        unsigned mine = n0, some = n0 > 0;
        for (int b = b0 + 1; b < b1; b++) {
            const int n = tiles_of<TILE>(span_of<ROWS>(p, b, flags));
            mine += n;
            some += n > 0;
        }
        const unsigned total = __reduce_add_sync(0xffffffffu, mine) * p.columns, there = __reduce_add_sync(0xffffffffu, some) * p.columns;
        size = max(MIN_TILES, (int)((float)total * p.per_cta));
        while ((unsigned)size * gridDim.x < total) size += 1 + (size >> 20);       // (the float is a little below the quotient)
        int unused = 0;
        if (DRAWS && B <= DRAWN_REQUESTS && size >= DRAWN_SHARE && there * 8 >= gridDim.x) {
            least = max(STAGES + 2, size / 64);
            unit = max(least, size / 16);
            size -= size / 8;
            drawn_from = size * (int)gridDim.x;
        } else if (there <= gridDim.x) {
            const int step = max(1, size / (CTAS > 1 ? 4 : 16)), most = CTAS > 1 ? size * EVEN_MOST / 8 + 2 : size + 2 * step;
#pragma unroll 1
            for (int tiles = size; tiles <= most; tiles += step) {
                even = __frcp_rn((float)tiles);
                unsigned k = parts_of(n0);
                for (int b = b0 + 1; b < b1; b++) k += parts_of(tiles_of<TILE>(span_of<ROWS>(p, b, unused)));
                if (__reduce_add_sync(0xffffffffu, k) * p.columns <= gridDim.x) {
                    mine = k;
                    break;
                }
                even = 0.0f;
            }
        }
        unsigned before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += u;
        }
        const unsigned all = __shfl_sync(0xffffffffu, before, 31) * p.columns;
        before -= mine;
        if (DRAWS && unit && warp == 0) {                   // (it is read behind the barriers at which pieces become known)
            unsigned tiles = before;
            for (int b = b0; b < b1; b++) { before_s[b] = tiles; tiles += tiles_of<TILE>(span_of<ROWS>(p, b, unused)); }
        }
        all_tiles = (int)all;
        r0 = (int)min((unsigned long long)all, (unsigned long long)(even != 0.0f ? 1 : size) * blockIdx.x);
        r1 = (int)min(all, (unsigned)r0 + (even != 0.0f ? 1 : size));
        // the lane that has the request of r0, and the request
        unsigned rest = (unsigned)r0 - before * p.columns;
        const bool here = (unsigned)r0 >= before * p.columns && rest < mine * p.columns;
        at.b = b0;
        if (here)
            for (; at.b < b1 - 1; at.b++) {
                const int n = tiles_of<TILE>(span_of<ROWS>(p, at.b, unused));
                const unsigned units = (unsigned)(even != 0.0f ? parts_of(n) : n) * p.columns;
                if (rest < units) break;
                rest -= units;
            }
        const int from = max(__ffs(__ballot_sync(0xffffffffu, here)) - 1, 0);
        at.b = min(__shfl_sync(0xffffffffu, at.b, from), B - 1);
        rest = __shfl_sync(0xffffffffu, rest, from);
        at.span = span_of<ROWS>(p, at.b, unused);
        at.n = tiles_of<TILE>(at.span);
        const int units = max(even != 0.0f ? parts_of(at.n) : at.n, 1);
        at.c = quotient((int)rest, units);
        at.i = (int)rest - at.c * units;                    // the tile, or the part
    }
    // rows without tokens, and those that are nobody's
    auto nothing = [&](int row) {
        if (KIND != WIDE_RESULTS) for (int i = tid; i < (int)a.Hq * (D / 8); i += THREADS)
            *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + row * a.out_token + i / (D / 8) * a.out_head + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
        if (a.lse) for (int h = tid; h < (int)a.Hq; h += THREADS) a.lse[row * a.Hq + h] = -CUDART_INF_F;
    };
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        if (tiles_of<TILE>(span_of<ROWS>(p, b, flags)) > 0) continue;
        if (KIND == WIDE_RESULTS) nothing(b);
        else for (int row = row_of<ROWS>(p, b), end = ROWS ? row_of<ROWS>(p, b + 1) : b + 1; row < end; row++) nothing(row);
    }
    if (ROWS && KIND != WIDE_RESULTS) for (int row = row_of<ROWS>(p, B) + (int)blockIdx.x; row < p.rows; row += (int)gridDim.x) nothing(row);
    // (in a call with prefixes what is ahead may still run, but not when this kernel has ended)
    auto behind = [&]() { if (KIND == WIDE_RESULTS && blockIdx.x == gridDim.x - 1) cudaGridDependencySynchronize(); };
    if (r0 >= r1) {
        behind();
        if (flags && a.status) atomicOr(a.status, flags);
        return;
    }

    // ---- the copies
    int share = r1 - r0, column_first = 0, parts = 1;       // column_first: the first CTA of this column's parts
    if (even != 0.0f) {                                     // part `i` of a column: the same number of tiles for each, the first ones have one more
        const int i = at.i;
        parts = parts_of(at.n);
        share = quotient(at.n, parts);
        const int more = at.n - share * parts;
        at.i = i * share + min(i, more);
        share += i < more;
        column_first = (int)blockIdx.x - i;
    }
    // pieces: the shares, then rounds of as many that are drawn, of half the size each time
    auto piece_of = [&](int tile) {
        if (!DRAWS || tile < drawn_from) return quotient(tile, size);
        int first = gridDim.x, tiles = unit;
        for (tile -= drawn_from; tiles > least && tile >= tiles * (int)gridDim.x; tiles = max(tiles / 2, least)) { tile -= tiles * (int)gridDim.x; first += gridDim.x; }
        return first + quotient(tile, tiles);
    };
    auto start_of = [&](int g, int &tiles) {
        tiles = size;
        if (!DRAWS || g < (int)gridDim.x) return g * size;
        int from = drawn_from;
        tiles = unit;
        for (g -= gridDim.x; tiles > least && g >= (int)gridDim.x; tiles = max(tiles / 2, least)) { from += tiles * (int)gridDim.x; g -= gridDim.x; }
        from += g * tiles;
        tiles = min(tiles, all_tiles - from);
        return from;
    };
    int piece = blockIdx.x, next = -1;                      // next: the piece behind this one, once it is known
    const int pieces_end = DRAWS && unit ? piece_of(all_tiles - 1) + 1 : 0;
    Place ahead = at;
    int to_copy = share;
    bool taken = false;                                     // `next` is being copied
    int page = -1;                                          // lanes 0 .. TOKENS - 1: the page of their token of the tile that is copied next
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * STAGE;
    auto ask = [&]() {
        page = -1;
        if (to_copy > 0 && lane < TOKENS) {
            const int t = ahead.span.first + ahead.i * TILE + warp % TEAM * TOKENS + lane;
            if (t < ahead.span.len) page = __ldg(a.table + ahead.b * a.table_stride + kvc_divide(t, p.page));
        }
    };
    auto copy_tile = [&](int stage) {
        if (to_copy > 0) {
            const int t = ahead.span.first + ahead.i * TILE + warp % TEAM * TOKENS + lane;
            const bool there = lane < TOKENS && t < ahead.span.len, good = there && (unsigned)page < p.n_pages;
            if (there && !good) flags |= KVC_FLAG_BAD_PAGE;
            const uint32_t mask = __ballot_sync(0xffffffffu, good);
            if (lane == 0) masks[warp][stage] = mask;
            if (mask) {
                const int hk = WH > 1 ? ahead.c * WH + warp / TEAM : (p.per_head == 1 ? ahead.c : ahead.c / p.per_head), row = t - kvc_divide(t, p.page) * (int)a.page_size;
                const Element *k16 = reinterpret_cast<const Element *>(a.kpages), *v16 = reinterpret_cast<const Element *>(a.vpages);
                if constexpr (CODED) {
                    const long long at = good ? page * p.s.k_page + hk * p.s.k_head + row : 0;
                    copy4(ring + stage * STAGE + 2 * HALF_STAGE + lane * 4, p.s.k + at, good);
                    copy4(ring + stage * STAGE + 2 * HALF_STAGE + TOKENS * 4 + lane * 4, p.s.v + at, good);
                }
                if (good) {
                    k16 += page * a.kp_page + row * (int)a.kp_row + hk * (int)a.kp_head;
                    if (!SAME) v16 += page * a.vp_page + row * (int)a.vp_row + hk * (int)a.vp_head;
                }
                const uint32_t to = ring + stage * STAGE;
                constexpr int PIECES = ROW / 16, SIDE = PIECES > 4 ? 8 : 4;                 // 16-byte pieces of a row, lanes that take a row's
                bool one_page = false;                      // (CODED) all of the tile's tokens are there and in one page: nobody has to be asked where his row is
                if constexpr (CODED) {
                    const int page0 = __shfl_sync(0xffffffffu, page, 0);
                    one_page = __all_sync(0xffffffffu, page == page0) && mask == ALL;
                    if (one_page) {
                        const uint8_t *k = reinterpret_cast<const uint8_t *>(a.kpages) + page0 * a.kp_page + __shfl_sync(0xffffffffu, row, 0) * (int)a.kp_row + hk * (int)a.kp_head + lane / SIDE * (int)a.kp_row +
                                           lane % SIDE * 16;
                        const int step = 32 / SIDE * (int)a.kp_row;
#pragma unroll
                        for (int j = 0; j < TOKENS * SIDE / 32; j++) {
#pragma unroll
                            for (int c = 0; c < (PIECES + SIDE - 1) / SIDE; c++) {
                                if (PIECES % SIDE == 0 || c * SIDE + lane % SIDE < PIECES) {
                                    const uint32_t at = to + piece_at<ROW>(32 / SIDE * j + lane / SIDE, c * SIDE + lane % SIDE);
                                    copy16(at, k + c * SIDE * 16, true);
                                    copy16(at + HALF_STAGE, k + c * SIDE * 16 + p.v_less_k, true);
                                }
                            }
                            k += step;
                        }
                    }
                }
                if (!one_page)
#pragma unroll
                for (int j = 0; j < TOKENS * SIDE / 32; j++) {
                    const int r = 32 / SIDE * j + lane / SIDE;
                    const bool on = mask >> r & 1;
                    const uint8_t *k = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k16), r)) + (lane % SIDE) * 16;
                    const uint8_t *v = SAME ? k + p.v_less_k : reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v16), r)) + (lane % SIDE) * 16;
#pragma unroll
                    for (int c = 0; c < (PIECES + SIDE - 1) / SIDE; c++) {
                        if (PIECES % SIDE == 0 || c * SIDE + lane % SIDE < PIECES) {
                            const uint32_t at = to + piece_at<ROW>(r, c * SIDE + lane % SIDE);
                            copy16(at, k + c * SIDE * 16, on);
                            copy16(at + HALF_STAGE, v + c * SIDE * 16, on);
                        }
                    }
                }
            }
            next_tile<TILE, ROWS>(p, ahead);
            if (--to_copy == 0 && DRAWS && next >= 0 && !taken) {
                const int tile = start_of(next, to_copy);
                int lo = 0, hi = B;
                while (hi - lo > 1) {                       // the last request with before_s * columns <= tile
                    const int mid = (lo + hi) >> 1;
                    if (before_s[mid] * p.columns <= (unsigned)tile) lo = mid; else hi = mid;
                }
                int unused = 0;
                const unsigned rest = (unsigned)tile - before_s[lo] * p.columns;
                ahead.b = lo;
                ahead.span = span_of<ROWS>(p, lo, unused);
                ahead.n = tiles_of<TILE>(ahead.span);
                ahead.c = quotient((int)rest, ahead.n);
                ahead.i = (int)rest - ahead.c * ahead.n;
                if (lane == 0) next_start_s[warp] = ahead;
                taken = true;
            }
        }
        copies_commit();
        ask();
    };

    // ---- the tiles
    uint32_t q[KS][NT][2];
    float o[KS][NT][4], m[NT][2], l[NT][2];
    int h0 = 0, heads = 0;
    float most[NT][2];                                      // (CODED) the largest product of a weight and a value's scale so far: the sums are lifted(most) times what they are
    float head_scale[NT][2];                                // (CODED, bf16) what the queries were divided by, of this lane's heads
    bool fresh = true;                                      // (CODED, bf16) the queries have not become fp16 yet
    auto begin_column = [&]() {                             // (the queries are asked for; they are first used behind the next wait)
        if (WH > 1) {
            h0 = (at.c * WH + warp / TEAM) * p.group;
            heads = p.group;
        } else {
            const int hk = p.per_head == 1 ? at.c : at.c / p.per_head, g = (int)(a.Hq / a.Hkv), sub = (at.c - hk * p.per_head) * p.group;
            h0 = hk * g + sub;
            heads = min(p.group, g - sub);
        }
        const int row = ROWS ? min(row_of<ROWS>(p, at.b), p.rows - 1) : at.b;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int h = nt * 8 + (lane >> 2);
            const T *from = reinterpret_cast<const T *>(a.q) + row * a.q_token + (h0 + h) * a.q_head + (lane & 3) * (CODED ? 4 : 2);
#pragma unroll
            for (int k = 0; k < KS; k++) {                  // (of codes a lane has four neighbours, as of the keys)
                q[k][nt][0] = h < heads ? *reinterpret_cast<const uint32_t *>(from + k * 16) : 0;
                q[k][nt][1] = h < heads ? *reinterpret_cast<const uint32_t *>(from + k * 16 + (CODED ? 2 : 8)) : 0;
            }
        }
        fresh = true;
    };
    auto to_half = [&]() {
        if constexpr (CODED && std::is_same_v<T, __nv_bfloat16>) {
            if (!fresh) return;
            fresh = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++) top = max(top, max(q[k][nt][e] & 0x7fffu, q[k][nt][e] >> 16 & 0x7fffu));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t exponent = max(top >> 7, 15u);                              // the largest value comes to lie in [2^14, 2^15)
                const float f = __uint_as_float((268 - exponent) << 23), back = __uint_as_float((exponent - 14) << 23);
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float2 v = Pair<T>::unpack(q[k][nt][e]);
                        q[k][nt][e] = Operand::pack(v.x * f, v.y * f);
                    }
#pragma unroll
                for (int e = 0; e < 2; e++) head_scale[nt][e] = __shfl_sync(0xffffffffu, back, ((lane & 3) * 2 + e) * 4);
            }
        }
    };
    auto clear = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int k = 0; k < KS; k++) o[k][nt][0] = o[k][nt][1] = o[k][nt][2] = o[k][nt][3] = 0.0f;
            m[nt][0] = m[nt][1] = -CUDART_INF_F;
            l[nt][0] = l[nt][1] = 0.0f;
            if (CODED) most[nt][0] = most[nt][1] = 0.0f;
        }
    };
    // where this lane's rows of a matrix load lie, from the stage's start: keys 16 rows by two pieces, values two pieces by 16 rows
    uint32_t key_at[4], value_at[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        key_at[k] = piece_at<ROW>(lane & 15, 2 * k + (lane >> 4));
        value_at[k] = HALF_STAGE + (CODED ? key_at[k] : piece_at<ROW>((lane & 7) + (lane >> 4) * 8, 2 * k + (lane >> 3 & 1)));      // (a piece of codes has 16 channels)
    }
    int stage = 0, first_i = at.i;                          // first_i: the first tile of the column that is this CTA's
    ask();
    begin_column();
    clear();
    int drawn = 0;
#pragma unroll 1
    for (int n = -STAGES;; n++) {                           // tile n of the piece
        if (n >= 0) {
            if (DRAWS && unit) {
                // The next piece is drawn as late as the copies allow: they are STAGES tiles ahead, and it takes a tile's time to know it.
                if (n == max(0, share - STAGES - 2) && tid == 0) drawn = atomicAdd(p.drawn, 1);
                if (n == max(min(1, share - 1), share - STAGES - 1)) {
                    if (tid == 0) {
                        next_s = (int)gridDim.x + drawn < pieces_end ? (int)gridDim.x + drawn : -1;
                        if (drawn == pieces_end - 1) *p.drawn = 0;                   // every CTA draws once in vain: this was the last of all
                    }
                    __syncthreads();
                    next = next_s;
                    taken = false;
                }
            }
            copies_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t mask = masks[warp][stage], from = ring + stage * STAGE;
            if constexpr (CODED) if (mask) {
                to_half();
                const float *const scales = reinterpret_cast<const float *>(smem + warp * STAGES * STAGE + stage * STAGE + 2 * HALF_STAGE);
                float s[2][NT][4];                          // of 16 tokens each
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float t[2][NT][4] = {};
#pragma unroll
                    for (int k = 0; k < KS / 2; k++) {
                        uint32_t f[4];
                        ldmatrix4(f, from + half * 16 * ROW + key_at[k & 3] + (k >> 2) * 128);
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t c0 = offset_codes<KIND, 1>(f[2 * j]), c1 = offset_codes<KIND, 1>(f[2 * j + 1]);
                            const uint32_t operand[4] = {two_codes<KIND, 0, 1>(c0), two_codes<KIND, 0, 1>(c1), two_codes<KIND, 2, 1>(c0), two_codes<KIND, 2, 1>(c1)};
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) Operand::mma(t[j][nt], operand, q[2 * k + j][nt][0], q[2 * k + j][nt][1]);
                        }
                    }
                    float k0 = scales[half * 16 + (lane >> 2)], k1 = scales[half * 16 + 8 + (lane >> 2)];
                    if (p.negative) k0 = -k0, k1 = -k1;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float back = e < 2 ? k0 : k1;
                            if constexpr (std::is_same_v<T, __nv_bfloat16>) back *= head_scale[nt][e & 1];      // (first: the products of codes and lifted queries may leave 32 bits with one of the two)
                            s[half][nt][e] = (t[0][nt][e] + t[1][nt][e]) * back;
                        }
                }
                if (mask != ALL) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const bool on0 = mask >> (half * 16 + (lane >> 2)) & 1, on1 = mask >> (half * 16 + 8 + (lane >> 2)) & 1;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) s[half][nt][e] = (e < 2 ? on0 : on1) ? s[half][nt][e] : -CUDART_INF_F;
                    }
                }
                float v[2][2], scale[NT][2], lift[NT][2];   // scales of this lane's tokens' values (left out ones have 0)
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int r = 0; r < 2; r++) v[half][r] = scales[TOKENS + half * 16 + 8 * r + (lane >> 2)];
                bool changes = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float largest[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) * p.log2_scaling;
                        top = fmaxf(top, m[nt][e]);
                        const float base = top == -CUDART_INF_F ? 0.0f : top;
                        scale[nt][e] = exp2_approx(m[nt][e] - base);
                        m[nt][e] = top;
#pragma unroll
                        for (int half = 0; half < 2; half++)
#pragma unroll
                            for (int i = e; i < 4; i += 2) s[half][nt][i] = exp2_approx(fmaf(s[half][nt][i], p.log2_scaling, -base));
                        l[nt][e] = fmaf(l[nt][e], scale[nt][e], (s[0][nt][e] + s[0][nt][e + 2]) + (s[1][nt][e] + s[1][nt][e + 2]));
#pragma unroll
                        for (int half = 0; half < 2; half++)
#pragma unroll
                            for (int r = 0; r < 2; r++) s[half][nt][e + 2 * r] *= v[half][r];
                        largest[e] = fmaxf(fmaxf(fabsf(s[0][nt][e]), fabsf(s[0][nt][e + 2])), fmaxf(fabsf(s[1][nt][e]), fabsf(s[1][nt][e + 2])));
                    }
                    uint32_t both = __byte_perm(__float_as_uint(largest[0]), __float_as_uint(largest[1]), 0x7632);      // (exponents are enough)
#pragma unroll
                    for (int i = 4; i < 32; i *= 2) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, i));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float before = lifted_back(most[nt][e]);
                        most[nt][e] = fmaxf(most[nt][e] * scale[nt][e], __uint_as_float(e ? both & 0xffff0000u : both << 16));
                        lift[nt][e] = lifted(most[nt][e]);
                        scale[nt][e] = scale[nt][e] * lift[nt][e] * before;                // (no more than 2: what it is the scale of was no more than `most`)
                        changes |= scale[nt][e] != 1.0f;
                    }
                }
                if (__any_sync(0xffffffffu, changes)) {
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            o[k][nt][0] *= scale[nt][0]; o[k][nt][1] *= scale[nt][1];
                            o[k][nt][2] *= scale[nt][0]; o[k][nt][3] *= scale[nt][1];
                        }
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const float w0 = s[half][nt][2 * e] * lift[nt][0], w1 = s[half][nt][2 * e + 1] * lift[nt][1];      // below 2^15
                            const uint32_t top = Operand::pack(w0, w1);
                            const float2 f = Operand::unpack(top);
                            hi[nt][e] = transpose8x8(top);
                            lo[nt][e] = transpose8x8(Operand::pack(w0 - f.x, w1 - f.y));
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KS / 2; k++) {
                        uint32_t f[4];
                        ldmatrix4_trans(f, from + half * 16 * ROW + value_at[k & 3] + (k >> 2) * 128);
#pragma unroll
                        for (int j = 0; j < 2; j++) {       // rows of the operand: even channels, odd ones
                            const uint32_t c0 = offset_codes<KIND, 2>(f[2 * j]), c1 = offset_codes<KIND, 2>(f[2 * j + 1]);
                            const uint32_t operand[4] = {two_codes<KIND, 0, 2>(c0), two_codes<KIND, 1, 2>(c0), two_codes<KIND, 0, 2>(c1), two_codes<KIND, 1, 2>(c1)};
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                Operand::mma(o[2 * k + j][nt], operand, hi[nt][0], hi[nt][1]);
                                Operand::mma(o[2 * k + j][nt], operand, lo[nt][0], lo[nt][1]);
                            }
                        }
                    }
                }
            }
            if constexpr (!CODED) if (mask) {
                float s[2][NT][4] = {};
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t f[4];
                    ldmatrix4(f, from + key_at[k & 3] + (k >> 2) * 128);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) Pair<T>::mma(s[k & 1][nt], f, q[k][nt][0], q[k][nt][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[0][nt][e] += s[1][nt][e];
                if (p.negative) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[0][nt][e] = -s[0][nt][e];
                }
                if (mask != ALL) {
                    const bool on0 = mask >> (lane >> 2) & 1, on1 = mask >> (8 + (lane >> 2)) & 1;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[0][nt][e] = (e < 2 ? on0 : on1) ? s[0][nt][e] : -CUDART_INF_F;
                }
                float scale[NT][2];
                bool grows = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) * p.log2_scaling;
                        top = fmaxf(top, m[nt][e]);
                        grows |= top > m[nt][e];
                        const float base = top == -CUDART_INF_F ? 0.0f : top;
                        scale[nt][e] = exp2_approx(m[nt][e] - base);
                        m[nt][e] = top;
                        s[0][nt][e] = exp2_approx(fmaf(s[0][nt][e], p.log2_scaling, LIFT - base));
                        s[0][nt][e + 2] = exp2_approx(fmaf(s[0][nt][e + 2], p.log2_scaling, LIFT - base));
                        l[nt][e] = fmaf(l[nt][e], scale[nt][e], s[0][nt][e] + s[0][nt][e + 2]);
                    }
                if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            o[k][nt][0] *= scale[nt][0]; o[k][nt][1] *= scale[nt][1];
                            o[k][nt][2] *= scale[nt][0]; o[k][nt][3] *= scale[nt][1];
                        }
                }
                uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t top = Pair<T>::pack(s[0][nt][2 * e], s[0][nt][2 * e + 1]);
                        const float2 f = Pair<T>::unpack(top);
                        hi[nt][e] = transpose8x8(top);
                        lo[nt][e] = transpose8x8(Pair<T>::pack(s[0][nt][2 * e] - f.x, s[0][nt][2 * e + 1] - f.y));
                    }
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t f[4];
                    ldmatrix4_trans(f, from + value_at[k & 3] + (k >> 2) * 128);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        Pair<T>::mma(o[k][nt], f, hi[nt][0], hi[nt][1]);
                        Pair<T>::mma(o[k][nt], f, lo[nt][0], lo[nt][1]);
                    }
                }
            }
            __syncwarp();                                   // everyone has read the stage
            if (at.i == at.n - 1 || n == share - 1) {
                // ---- the column's end in this share: the warps' results are joined; the stage just read holds their sums meanwhile
                const uint32_t scratch = stage * STAGE;
                if constexpr (CODED) {                      // what was taken out of the sums
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const float back[2] = {lifted_back(most[nt][0]), lifted_back(most[nt][1])};
#pragma unroll
                        for (int k = 0; k < KS; k++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[k][nt][e] *= back[e & 1];
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float v = l[nt][e];
                        v += __shfl_xor_sync(0xffffffffu, v, 4);
                        v += __shfl_xor_sync(0xffffffffu, v, 8);
                        v += __shfl_xor_sync(0xffffffffu, v, 16);
                        const int h = nt * 8 + (lane & 3) * 2 + e;
                        if (lane < 4) ml_s[warp][h] = make_float2(m[nt][e], v);
                        if (h < heads) {
                            float *to = reinterpret_cast<float *>(smem + warp * STAGES * STAGE + scratch) + h * D;
#pragma unroll
                            for (int k = 0; k < KS; k++) {
                                if constexpr (CODED) {
                                    *reinterpret_cast<float2 *>(to + ((k * 16 + 2 * (lane >> 2)) ^ ((h >> 1 & 3) * 8))) = make_float2(o[k][nt][e], o[k][nt][e + 2]);
                                } else {
                                    to[(k * 16 + (lane >> 2)) ^ ((h >> 1 & 3) * 8)] = o[k][nt][e];
                                    to[(k * 16 + 8 + (lane >> 2)) ^ ((h >> 1 & 3) * 8)] = o[k][nt][e + 2];
                                }
                            }
                        }
                    }
                const int of_b = at.b, of_row = KIND == WIDE_RESULTS ? at.b : ROWS ? min(row_of<ROWS>(p, at.b), p.rows - 1) : at.b, of_h0 = WH > 1 ? at.c * WH * p.group : h0, of_heads = WH * heads, pieces = of_heads * (D / 4);      // of all its KV heads
                const bool whole = first_i == 0 && at.i == at.n - 1;        // the column lies in this share
                const int begin = r0 + n - at.i;            // its first tile in the row of tiles
                const int tiles = at.n, of_piece = piece, place = 2 * piece + (n - (at.i - first_i) > 0);
                first_i = 0;
                if (n < share - 1) {
                    next_tile<TILE, ROWS>(p, at);
                } else if (DRAWS && next >= 0) {
                    piece = next;
                    next = -1;
                    r0 = start_of(piece, share);
                    at = next_start_s[warp];
                    first_i = at.i;
                    n = -1;                                 // (the loop goes on with 0)
                } else n = share;                           // (it ends)
                if (n != share) begin_column();             // on their way while the sums are joined
                clear();
                __syncthreads();
                unsigned odd = 0;                           // query heads whose result has channels that are no numbers although its weights are: a bit for each
                auto write = [&](int i, float top, float sum, const float4 &v) {       // four channels of a result
                    const int h = of_h0 + i / (D / 4), d = i % (D / 4) * 4;
                    const float f = sum == 0.0f ? 0.0f : 1.0f / sum, any = v.x + v.y + v.z + v.w;
                    if (!CODED && KIND != WIDE_RESULTS) odd |= any != any && sum == sum ? 1u << (h - of_h0) : 0;
                    if constexpr (KIND == WIDE_RESULTS) __stcg(reinterpret_cast<float4 *>(p.wide + ((long long)of_row * a.Hq + h) * D + d), make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
                    else *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + of_row * a.out_token + h * a.out_head + d) =
                        make_uint2(Pair<T>::pack(v.x * f, v.y * f), Pair<T>::pack(v.z * f, v.w * f));
                    if (d == 0 && a.lse) a.lse[of_row * a.Hq + h] = sum == 0.0f ? -CUDART_INF_F : (top + log2f(sum) - LIFT) * 0.69314718055994531f;
                };
                float *part = p.parts + (long long)place * p.part;
                // the warps of a KV head join their sums
                const int mine = of_heads / WH, sub = warp / TEAM * mine;       // a KV head's query heads, the first of them among the column's
                for (int i = tid % (TEAM * 32); i < mine * (D / 4); i += TEAM * 32) {
                    const int h = i / (D / 4), d = i % (D / 4) * 4;
                    float2 ml[TEAM];
                    float top = -CUDART_INF_F, sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < TEAM; w++) { ml[w] = ml_s[warp / TEAM * TEAM + w][h]; top = fmaxf(top, ml[w].x); }
                    const float base = top == -CUDART_INF_F ? 0.0f : top;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < TEAM; w++) {
                        const float f = exp2_approx(ml[w].x - base);
                        const float4 x = *reinterpret_cast<const float4 *>(smem + (warp / TEAM * TEAM + w) * STAGES * STAGE + scratch + (h * D + (d ^ ((h >> 1 & 3) * 8))) * 4);
                        sum += f * ml[w].y;
                        v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
                    }
                    if (whole) write(sub * (D / 4) + i, top, sum, v);
                    else {
                        __stcg(reinterpret_cast<float4 *>(part) + sub * (D / 4) + i, v);
                        if (d == 0) __stcg(reinterpret_cast<float2 *>(part + WH * p.group * D) + sub + h, make_float2(top, sum));
                    }
                }
                if (odd) odd_s = 1;
                __syncthreads();
                if (!whole) {
                    const int w_first = even != 0.0f ? column_first : piece_of(begin), count = even != 0.0f ? parts : piece_of(begin + tiles - 1) - w_first + 1;
                    int unused;
                    const int first_place = 2 * w_first + (even == 0.0f && begin > start_of(w_first, unused));
                    float4 *const join_v = reinterpret_cast<float4 *>(smem + scratch);       // (the stage that held the sums)
                    float2 *const join_ml = reinterpret_cast<float2 *>(join_v + THREADS);
                    static_assert(THREADS * 24 <= STAGE && MAX_GROUP * D + 4 <= STAGE && WH * D / 8 <= 32, "a stage has room for what is joined, and for what infinite_values keeps");
                    // the results of every step-th of `many` pieces from w on become one: the column's, or one in the first of their places
                    auto join = [&](int w, int step, int many, bool final) {
                        const int per = min(pieces, THREADS), ways = THREADS / per, way = tid / per;
                        for (int i = tid - way * per; i < pieces; i += per) {
                            const int h = i / (D / 4);
                            float top = -CUDART_INF_F, sum = 0.0f;
                            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (way < ways) {
                                for (int u0 = way; u0 < many; u0 += JOINED * ways) {
                                    float2 ml[JOINED];
                                    float4 x[JOINED];
#pragma unroll
                                    for (int k = 0; k < JOINED; k++) {
                                        const int u = u0 + k * ways, from_w = w + u * step;
                                        const float *from = p.parts + (long long)(from_w == w_first ? first_place : 2 * from_w) * p.part;
                                        ml[k] = make_float2(-CUDART_INF_F, 0.0f);
                                        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                        if (u < many) {
                                            ml[k] = __ldcg(reinterpret_cast<const float2 *>(from + WH * p.group * D) + h);
                                            x[k] = __ldcg(reinterpret_cast<const float4 *>(from) + i);
                                        }
                                    }
                                    float now = top;
#pragma unroll
                                    for (int k = 0; k < JOINED; k++) now = fmaxf(now, ml[k].x);
                                    const float base = now == -CUDART_INF_F ? 0.0f : now, f = exp2_approx(top - base);
                                    sum *= f; v.x *= f; v.y *= f; v.z *= f; v.w *= f;
#pragma unroll
                                    for (int k = 0; k < JOINED; k++) {
                                        const float g = exp2_approx(ml[k].x - base);
                                        sum += ml[k].y * g;
                                        v.x += x[k].x * g; v.y += x[k].y * g; v.z += x[k].z * g; v.w += x[k].w * g;
                                    }
                                    top = now;
                                }
                            }
                            if (ways > 1) {                 // (the loop is entered once then)
                                join_v[tid] = v;
                                join_ml[tid] = make_float2(top, sum);
                                __syncthreads();
                                if (tid >= pieces) continue;
                                top = -CUDART_INF_F; sum = 0.0f;
                                v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                for (int k = 0; k < ways; k++) top = fmaxf(top, join_ml[k * per + tid].x);
                                const float base = top == -CUDART_INF_F ? 0.0f : top;
                                for (int k = 0; k < ways; k++) {
                                    const float2 ml = join_ml[k * per + tid];
                                    const float4 x = join_v[k * per + tid];
                                    const float g = exp2_approx(ml.x - base);
                                    sum += ml.y * g;
                                    v.x += x.x * g; v.y += x.y * g; v.z += x.z * g; v.w += x.w * g;
                                }
                            } else if (way >= ways) continue;
                            if (final) write(i, top, sum, v);
                            else {                          // (others may still read the maxima and sums there)
                                __stcg(reinterpret_cast<float4 *>(p.parts + (long long)(w == w_first ? first_place : 2 * w) * p.part) + i, v);
                                if (i % (D / 4) == 0) new_ml[h] = make_float2(top, sum);
                            }
                        }
                        if (odd) odd_s = 1;
                        __syncthreads();
                        if (!final) {
                            if (tid < of_heads) __stcg(reinterpret_cast<float2 *>(p.parts + (long long)(w == w_first ? first_place : 2 * w) * p.part + WH * p.group * D) + tid, new_ml[tid]);
                            __syncthreads();
                        }
                    };
                    // whether this CTA is the last of `many` at a counter, which is zero again then; what they wrote before is seen behind it
                    auto is_last = [&](unsigned *counter, int many) {
                        if (tid == 0) {
                            unsigned before;                // (the barrier ahead made the CTA's writes this thread's: it releases them, and acquires the others')
                            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                            const bool last = before == (unsigned)(many - 1);
                            if (last) *counter = 0;
                            last_s = last;
                        }
                        __syncthreads();
                        const bool last = last_s;
                        __syncthreads();
                        return last;
                    };
                    // Few parts are joined at once; many by eights first, each eight by the last of them: one trip to memory for eight results
                    // at a time.
                    if (count <= 2 * JOINED) {
                        if (is_last(p.counters + first_place, count)) join(w_first, 1, count, true);
                    } else {
                        const int g = (of_piece - w_first) / JOINED, leader = w_first + g * JOINED, groups = (count + JOINED - 1) / JOINED, many = min(JOINED, count - g * JOINED);
                        if (is_last(p.group_counters + (leader == w_first ? first_place : 2 * leader), many)) {
                            join(leader, 1, many, false);
                            if (is_last(p.counters + first_place, groups)) join(w_first, JOINED, groups, true);
                        }
                    }
                }
                if constexpr (!CODED && KIND != WIDE_RESULTS) if (odd_s) {      // (of 256 requests of 64 tokens, a column of one tile, asking takes 0.5 of 17.6 us, 8 x 4096 84.6 with and without)
                    __syncthreads();
                    if (tid == 0) odd_s = 0;
                    __syncthreads();
                    if (odd) atomicOr(&odd_s, odd);
                    __syncthreads();
                    infinite_values<T, D, ROWS>(p, of_b, of_row, of_h0, of_heads, odd_s, reinterpret_cast<uint32_t *>(smem + scratch));
                    if (tid == 0) odd_s = 0;
                }
            } else {
                at.i++;
            }
        }
        if (n == share) break;
        // the stage that was read is filled again; nothing is read in the first rounds
        copy_tile(stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    copies_wait<0>();
    behind();
    if (flags && a.status) atomicOr(a.status, flags);
}

// ROWS is a kernel of its own: asked in the kernel, whether there are `starts` took 0.9 of 37 us of calls without any (76 requests of up to 2014 tokens, 10 KV heads of 64
// channels).  With ROWS a call takes 0.1 to 0.7 us more (777 tokens of 32 heads 8.4 and 8.6, 8 x 4096 84.6 and 85.3), of 256 requests of 64 tokens 17.0 and 18.7.
template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS, bool ROWS, int KIND>
int launch_kernel(Params &p, cudaStream_t stream) {
    static kvc_launch_slot slot;
    constexpr size_t shared = (size_t)WARPS * STAGES * Tiles<D, KIND>::STAGE;
    auto *kernel = paged_attn_kernel<T, D, NT, WH, SAME, STAGES, CTAS, ROWS, KIND>;
    int occ = 0;
    if (int rc = kvc_prepare(slot, reinterpret_cast<const void *>(kernel), THREADS, shared, &occ)) return rc;
    KVC_REQUIRE(occ > 0, "kvc_paged_attn: the kernel does not fit this device");
    constexpr int TILE = Tiles<D, KIND>::TOKENS * WARPS / WH;
    p.columns /= WH;
    const long long most_tiles = p.a.B * p.columns * ((p.a.table_width * p.a.page_size + TILE - 1) / TILE);
    KVC_REQUIRE(p.a.B * p.columns < (1ll << 31) && most_tiles < (1ll << 31) - (1 << 20), "kvc_paged_attn: requests, KV heads and table rows of more than 2^31 tiles of %d tokens", TILE);
    const long long grid = std::max<long long>(std::min<long long>(most_tiles, (long long)std::min(occ, MAX_CTAS_PER_SM) * kvc_sm_count()), 1);
    p.per_cta = (float)(0.9999997 / grid);
    if (KIND == WIDE_RESULTS) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = shared;
        cfg.stream = stream;
        cudaLaunchAttribute early;
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        KVC_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, (const Params)p));
        return KVC_OK;
    }
    kernel<<<(unsigned)grid, THREADS, shared, stream>>>(p);
    KVC_LAUNCH_OK();
    return KVC_OK;
}

template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS, int KIND = 0>
int launch(Params &p, cudaStream_t s) {
    return p.starts ? launch_kernel<T, D, NT, WH, SAME, STAGES, CTAS, true, KIND>(p, s) : launch_kernel<T, D, NT, WH, SAME, STAGES, CTAS, false, KIND>(p, s);
}

// the kernels for rows of codes, and those with results of 32 bits (files of their own: they take as long to compile as the others)
int launch_codes(Params &p, cudaStream_t s);
int launch_wide(Params &p, cudaStream_t s);

// query heads that a column takes at most: 16 where they fit the registers beside the accumulators
inline int group_of(int64_t Hq, int64_t Hkv, int64_t D) { return (int)std::min<int64_t>(Hq / Hkv, D > 128 ? 8 : MAX_GROUP); }
inline int64_t columns_of(int64_t Hq, int64_t Hkv, int64_t D) { return Hkv * ((Hq / Hkv + group_of(Hq, Hkv, D) - 1) / group_of(Hq, Hkv, D)); }
// Of partial results: two for every piece.  Of s tiles for a CTA s / 8 and those left by rounding down are drawn, in rounds of s / 16, s / 32, s / 64 (at least) and what these leave:
// a CTA's share and five pieces more.
inline int64_t places(int64_t D) { return 2ll * 6 * (D == 64 ? 4 : 3) * kvc_sm_count(); }
// Floats of a place: of two KV heads where they are read together; room for eight heads at least, so that one workspace serves more shapes.  A multiple of four: values are
// written and read sixteen bytes at a time, and n (D + 2) is two more than one for odd n.
inline int64_t part_floats(int64_t group, int64_t D) { return (std::max<int64_t>(group <= 8 && D < 128 ? 2 * group : group, 8) * (D + 2) + 3) / 4 * 4; }
// The counter of what is drawn, and two counters for a place: of the column whose first result lies there, of the eight results that begin there.  They lie in
// front, the same for calls of all shapes: a workspace may serve one after the other.
inline int64_t counter_bytes() { return 256 + (2 * places(64) * 4 + 255) / 256 * 256; }

// Strides and places of rows, asked alike by all entries (name: which): rows start on 16 bytes, those of pools on `elements`, and a row's place in its page is a number of 32 bits.  The
// stride of a dimension of one may be anything, and becomes 0.
inline int check_rows(kvc_paged_attn_args &a, int64_t rows, int64_t elements, const char *name) {
    if (a.Hq == 1) a.q_head = a.out_head = 0;
    if (rows == 1) a.q_token = a.out_token = 0;
    if (a.Hkv == 1) a.kp_head = a.vp_head = 0;
    if (a.page_size == 1) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1) a.kp_page = a.vp_page = 0;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages) | reinterpret_cast<uintptr_t>(a.out);
    const int64_t strides = a.q_token | a.q_head | a.out_token | a.out_head, of_pools = a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head;
    KVC_REQUIRE((at & 15) == 0 && (strides & 7) == 0 && (of_pools & (elements - 1)) == 0, "%s: rows must start on 16 bytes", name);
    const int64_t last = a.page_size - 1, head = a.Hkv - 1, most = 1ll << 31;              // (each product by itself first: their sum is one of 64 bits then)
    KVC_REQUIRE(a.kp_row >= 0 && a.kp_head >= 0 && a.vp_row >= 0 && a.vp_head >= 0 && a.kp_page >= 0 && a.vp_page >= 0, "%s: the pools have a negative stride", name);
    KVC_REQUIRE(a.kp_row < most && a.kp_head < most && a.vp_row < most && a.vp_head < most && a.kp_row * last + a.kp_head * head < most && a.vp_row * last + a.vp_head * head < most,
                "%s: a page spans more than 2^31 elements", name);
    return KVC_OK;
}
// Results overlap neither one another nor queries that they are not.
inline int check_results(const kvc_paged_attn_args &a, int64_t rows, const char *name) {
    const kvc_rows q = kvc_make_rows(a.q, a.D, rows, a.q_token, a.Hq, a.q_head), out = kvc_make_rows(a.out, a.D, rows, a.out_token, a.Hq, a.out_head);
    KVC_REQUIRE(out.apart, "%s: rows of the output overlap", name);
    KVC_REQUIRE(kvc_rows_equal(q, out) || !kvc_rows_overlap(q, out), "%s: the output overlaps the queries and is not them", name);
    return KVC_OK;
}

// What a call's arguments say, for a kernel: sizes have been checked.
inline void set_params(Params &p, const kvc_paged_attn_args &a, const int32_t *starts, int64_t rows) {
    p.a = a;
    p.page = kvc_make_div((uint32_t)a.page_size);
    p.group = group_of(a.Hq, a.Hkv, a.D);
    p.columns = (int)columns_of(a.Hq, a.Hkv, a.D);
    p.per_head = p.columns / (int)a.Hkv;
    p.chunk = (int)((a.B + 31) / 32);
    p.most_tokens = (int)(a.table_width * a.page_size);
    p.n_pages = (unsigned)a.n_pages;
    p.starts = starts;
    p.rows = (int)rows;
    p.negative = a.scaling < 0.0f;
    p.log2_scaling = std::max(fabsf(a.scaling) * 1.4426950408889634f, 1e-37f);      // (0 times the -inf of a token that is left out is none)
    p.part = (int)part_floats(p.group, a.D);
    p.drawn = reinterpret_cast<int *>(a.workspace);
    p.counters = reinterpret_cast<unsigned *>(a.workspace) + 64;
    p.group_counters = p.counters + places(64);
    p.parts = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(a.workspace) + counter_bytes());
    p.v_less_k = reinterpret_cast<const uint8_t *>(a.vpages) - reinterpret_cast<const uint8_t *>(a.kpages);
}

}  // namespace kvc_paged

