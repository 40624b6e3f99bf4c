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
#include <math_constants.h>
#include <string.h>

#include <algorithm>

#include "kvc_paged.cuh"

namespace {

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

// where a 16-byte piece of a row lies in a stage: the 8 rows of a matrix load fall on different banks
template <int D> __device__ __forceinline__ uint32_t piece_at(int row, int piece) {
    if constexpr (D % 64 == 0) return (uint32_t)(row * (D / 8) + (piece ^ (row & 7))) * 16;       // rows start on bank 0
    else return (uint32_t)(row * (D / 8) + (piece ^ ((row >> 1) & 3))) * 16;                        // D = 96: every other row starts in the middle
}

// The first of a request's rows of q and out, for b = B the first that is nobody's.  (Kept inside the tensors whatever `starts` hold, as lengths are.)
template <bool ROWS> __device__ __forceinline__ int row_of(const Params &p, int b) { return ROWS ? min(max(p.starts[b], 0), p.rows) : b; }

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

template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS, bool ROWS>
__global__ void __launch_bounds__(THREADS, CTAS) paged_attn_kernel(const __grid_constant__ Params p) {
    constexpr int KS = D / 16;                              // steps of 16 channels
    constexpr int TEAM = WARPS / WH, TILE = 16 * TEAM;      // warps of a KV head, tokens of a tile
    constexpr uint32_t HALF_STAGE = 16 * D * 2, STAGE = 2 * HALF_STAGE;
    constexpr float LIFT = Pair<T>::LIFT;
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
    // shares 19.6, 49.4, 90).  Tiles of shorter rows are less to have under way: 5 / 4 (11 x 4096 tokens of 32 heads of 96 channels 94 us, with 7 / 4 99); where an SM
    // holds one CTA, 9 / 8.  Else equal shares of the row of all columns' tiles.
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
            const int step = max(1, size / (CTAS > 1 ? 4 : 16)), most = CTAS > 1 ? size * (D < 128 ? 5 : 7) / 4 + 2 : size + 2 * step;
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
        for (int i = tid; i < (int)a.Hq * (D / 8); i += THREADS)
            *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + row * a.out_token + i / (D / 8) * a.out_head + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
        if (a.lse) for (int h = tid; h < (int)a.Hq; h += THREADS) a.lse[row * a.Hq + h] = -CUDART_INF_F;
    };
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        if (tiles_of<TILE>(span_of<ROWS>(p, b, flags)) > 0) continue;
        for (int row = row_of<ROWS>(p, b), end = ROWS ? row_of<ROWS>(p, b + 1) : b + 1; row < end; row++) nothing(row);
    }
    if (ROWS) for (int row = row_of<ROWS>(p, B) + (int)blockIdx.x; row < p.rows; row += (int)gridDim.x) nothing(row);
    if (r0 >= r1) {
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
    int page = -1;                                          // lanes 0 .. 15: the page of their token of the tile that is copied next
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * STAGE;
    auto ask = [&]() {
        page = -1;
        if (to_copy > 0 && lane < 16) {
            const int t = ahead.span.first + ahead.i * TILE + warp % TEAM * 16 + lane;
            if (t < ahead.span.len) page = __ldg(a.table + ahead.b * a.table_stride + kvc_divide(t, p.page));
        }
    };
    auto copy_tile = [&](int stage) {
        if (to_copy > 0) {
            const int t = ahead.span.first + ahead.i * TILE + warp % TEAM * 16 + lane;
            const bool there = lane < 16 && t < ahead.span.len, good = there && (unsigned)page < p.n_pages;
            if (there && !good) flags |= KVC_FLAG_BAD_PAGE;
            const uint32_t mask = __ballot_sync(0xffffffffu, good);
            if (lane == 0) masks[warp][stage] = mask;
            if (mask) {
                const int hk = WH > 1 ? ahead.c * WH + warp / TEAM : (p.per_head == 1 ? ahead.c : ahead.c / p.per_head), row = t - kvc_divide(t, p.page) * (int)a.page_size;
                const T *k16 = reinterpret_cast<const T *>(a.kpages), *v16 = reinterpret_cast<const T *>(a.vpages);
                if (good) {
                    k16 += page * a.kp_page + row * (int)a.kp_row + hk * (int)a.kp_head;
                    if (!SAME) v16 += page * a.vp_page + row * (int)a.vp_row + hk * (int)a.vp_head;
                }
                const uint32_t to = ring + stage * STAGE;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = 4 * j + (lane >> 3);
                    const bool on = mask >> r & 1;
                    const uint8_t *k = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k16), r)) + (lane & 7) * 16;
                    const uint8_t *v = SAME ? k + p.v_less_k : reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v16), r)) + (lane & 7) * 16;
#pragma unroll
                    for (int c = 0; c < (D / 8 + 7) / 8; c++) {
                        if ((D / 8) % 8 == 0 || c * 8 + (lane & 7) < D / 8) {
                            const uint32_t at = to + piece_at<D>(r, c * 8 + (lane & 7));
                            copy16(at, k + c * 128, on);
                            copy16(at + HALF_STAGE, v + c * 128, on);
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
            const T *from = reinterpret_cast<const T *>(a.q) + row * a.q_token + (h0 + h) * a.q_head + (lane & 3) * 2;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                q[k][nt][0] = h < heads ? *reinterpret_cast<const uint32_t *>(from + k * 16) : 0;
                q[k][nt][1] = h < heads ? *reinterpret_cast<const uint32_t *>(from + k * 16 + 8) : 0;
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
        }
    };
    // where this lane's rows of a matrix load lie, from the stage's start: keys 16 rows by two pieces, values two pieces by 16 rows
    uint32_t key_at[4], value_at[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        key_at[k] = piece_at<D>(lane & 15, 2 * k + (lane >> 4));
        value_at[k] = HALF_STAGE + piece_at<D>((lane & 7) + (lane >> 4) * 8, 2 * k + (lane >> 3 & 1));
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
            if (mask) {
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
                if (mask != 0xffff) {
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
                                to[(k * 16 + (lane >> 2)) ^ ((h >> 1 & 3) * 8)] = o[k][nt][e];
                                to[(k * 16 + 8 + (lane >> 2)) ^ ((h >> 1 & 3) * 8)] = o[k][nt][e + 2];
                            }
                        }
                    }
                const int of_b = at.b, of_row = ROWS ? min(row_of<ROWS>(p, at.b), p.rows - 1) : at.b, of_h0 = WH > 1 ? at.c * WH * p.group : h0, of_heads = WH * heads, pieces = of_heads * (D / 4);      // of all its KV heads
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
                    odd |= any != any && sum == sum ? 1u << (h - of_h0) : 0;
                    *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + of_row * a.out_token + h * a.out_head + d) =
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
                if (odd_s) {                                // (of 256 requests of 64 tokens, a column of one tile, asking takes 0.5 of 17.6 us, 8 x 4096 84.6 with and without)
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
    if (flags && a.status) atomicOr(a.status, flags);
}

// ROWS is a kernel of its own: asked in the kernel, whether there are `starts` took 0.9 of 37 us of calls without any (76 requests of up to 2014 tokens, 10 KV heads of 64
// channels).  With ROWS a call takes 0.1 to 0.7 us more (777 tokens of 32 heads 8.4 and 8.6, 8 x 4096 84.6 and 85.3), of 256 requests of 64 tokens 17.0 and 18.7.
template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS, bool ROWS>
int launch_kernel(Params &p, cudaStream_t stream) {
    static kvc_launch_slot slot;
    constexpr size_t shared = (size_t)WARPS * STAGES * 64 * D;
    auto *kernel = paged_attn_kernel<T, D, NT, WH, SAME, STAGES, CTAS, ROWS>;
    int occ = 0;
    if (int rc = kvc_prepare(slot, reinterpret_cast<const void *>(kernel), THREADS, shared, &occ)) return rc;
    KVC_REQUIRE(occ > 0, "kvc_paged_attn: the kernel does not fit this device");
    constexpr int TILE = 16 * WARPS / WH;
    p.columns /= WH;
    const long long most_tiles = p.a.B * p.columns * ((p.a.table_width * p.a.page_size + TILE - 1) / TILE);
    KVC_REQUIRE(p.a.B * p.columns < (1ll << 31) && most_tiles < (1ll << 31) - (1 << 20), "kvc_paged_attn: requests, KV heads and table rows of more than 2^31 tiles of %d tokens", TILE);
    const long long grid = std::max<long long>(std::min<long long>(most_tiles, (long long)std::min(occ, MAX_CTAS_PER_SM) * kvc_sm_count()), 1);
    p.per_cta = (float)(0.9999997 / grid);
    kernel<<<(unsigned)grid, THREADS, shared, stream>>>(p);
    KVC_LAUNCH_OK();
    return KVC_OK;
}

template <typename T, int D, int NT, int WH, bool SAME, int STAGES, int CTAS>
int launch(Params &p, cudaStream_t s) {
    return p.starts ? launch_kernel<T, D, NT, WH, SAME, STAGES, CTAS, true>(p, s) : launch_kernel<T, D, NT, WH, SAME, STAGES, CTAS, false>(p, s);
}

// Stages of a warp's ring and CTAs of an SM, for up to 8 query heads of a KV head and for up to 16 (their accumulators take the registers of the third CTA): as many copies
// under way as the shared memory holds.  128 channels: three CTAs of two stages, 89.5 us for 8 x 4096 tokens of 32 heads and 33.5 for 256 requests of up to 300,
// two of three 95.5 and 46.8.
template <typename T, int D, int STAGES, int CTAS, int WIDE_STAGES, int WIDE_CTAS>
int choose_heads(Params &p, bool same, cudaStream_t s) {
    if constexpr (WIDE_STAGES > 0) {
        if (p.group > 8) return same ? launch<T, D, 2, 1, true, WIDE_STAGES, WIDE_CTAS>(p, s) : launch<T, D, 2, 1, false, WIDE_STAGES, WIDE_CTAS>(p, s);
    }
    // Rows of 64 and 96 channels that lie head by head behind one another leave half of what the memory delivers at a time to the neighbour's row: two KV heads are read
    // together.  32 x 8192 tokens of 8 heads: of 96 channels 134 us, 177 one by one, of 64 89.5 and 91.4; 11 x 4096 of 32 heads of 96 94 and 126.  (Of 128: 326 and 317 us
    // for 16 x 32768.)
    if constexpr (D < 128) {
        if (same && p.per_head == 1 && p.a.Hkv % 2 == 0 && p.a.kp_head < p.a.kp_row) return launch<T, D, 1, 2, true, STAGES, CTAS>(p, s);
    }
    return same ? launch<T, D, 1, 1, true, STAGES, CTAS>(p, s) : launch<T, D, 1, 1, false, STAGES, CTAS>(p, s);
}

template <typename T>
int choose(Params &p, bool same, cudaStream_t s) {
    switch (p.a.D) {
        case 64: return choose_heads<T, 64, 3, 4, 4, 3>(p, same, s);
        case 96: return choose_heads<T, 96, 3, 3, 4, 2>(p, same, s);
        case 128: return choose_heads<T, 128, 2, 3, 3, 2>(p, same, s);
        default: return choose_heads<T, 256, 3, 1, 0, 0>(p, same, s);
    }
}

// query heads that a column takes at most: 16 where they fit the registers beside the accumulators
int group_of(int64_t Hq, int64_t Hkv, int64_t D) { return (int)std::min<int64_t>(Hq / Hkv, D > 128 ? 8 : MAX_GROUP); }
int64_t columns_of(int64_t Hq, int64_t Hkv, int64_t D) { return Hkv * ((Hq / Hkv + group_of(Hq, Hkv, D) - 1) / group_of(Hq, Hkv, D)); }
// Of partial results: two for every piece.  Of s tiles for a CTA s / 8 and those left by rounding down are drawn, in rounds of s / 16, s / 32, s / 64 (at least) and what these leave:
// a CTA's share and five pieces more.
int64_t places(int64_t D) { return 2ll * 6 * (D == 64 ? 4 : 3) * kvc_sm_count(); }
// Floats of a place: of two KV heads where they are read together; room for eight heads at least, so that one workspace serves more shapes.  A multiple of four: values are
// written and read sixteen bytes at a time, and n (D + 2) is two more than one for odd n.
int64_t part_floats(int64_t group, int64_t D) { return (std::max<int64_t>(group <= 8 && D < 128 ? 2 * group : group, 8) * (D + 2) + 3) / 4 * 4; }
// The counter of what is drawn, and two counters for a place: of the column whose first result lies there, of the eight results that begin there.  They lie in
// front, the same for calls of all shapes: a workspace may serve one after the other.
int64_t counter_bytes() { return 256 + (2 * places(64) * 4 + 255) / 256 * 256; }

}  // namespace

extern "C" int64_t kvc_paged_attn_cleared(void) { return counter_bytes(); }
extern "C" int64_t kvc_paged_attn_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    if (B < 0 || Hkv <= 0 || Hq < Hkv || D <= 0) return 0;
    return counter_bytes() + places(D) * part_floats(group_of(Hq, Hkv, D), D) * 4;
}

// starts null: a row for each request
static int paged_attn(const kvc_paged_attn_args *args, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_paged_attn: null pointer");
    kvc_paged_attn_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_paged_attn: unknown type %d", a.type);
    KVC_REQUIRE(a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256, "kvc_paged_attn: heads of 64, 96, 128 or 256 channels, got %lld", (long long)a.D);
    KVC_REQUIRE(a.B >= 0 && a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0 && a.Hq < 65536, "kvc_paged_attn: %lld query heads over %lld", (long long)a.Hq, (long long)a.Hkv);
    KVC_REQUIRE(a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages >= 0 && a.n_pages < (1ll << 31) && a.table_width >= 0 && a.window >= 0, "kvc_paged_attn: bad sizes");
    KVC_REQUIRE(a.table_width * a.page_size < (1ll << 31) - 256, "kvc_paged_attn: a table row holds %lld tokens, lengths have 32 bits", (long long)(a.table_width * a.page_size));
    if (!starts) rows = a.B;
    KVC_REQUIRE(rows >= 0 && rows < (1 << 24) && (a.B > 0 || rows == 0), "kvc_paged_attn: %lld rows of %lld requests", (long long)rows, (long long)a.B);
    if (rows == 0) return KVC_OK;
    KVC_REQUIRE(a.B < (1 << 24), "kvc_paged_attn: %lld requests", (long long)a.B);
    KVC_REQUIRE(a.q && a.out && a.lengths && (a.table || a.table_width == 0) && ((a.kpages && a.vpages) || a.n_pages == 0), "kvc_paged_attn: null pointer");
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages) | reinterpret_cast<uintptr_t>(a.out);
    if (a.Hq == 1) a.q_head = a.out_head = 0;              // (the stride of a dimension of one may be anything)
    if (rows == 1) a.q_token = a.out_token = 0;
    if (a.Hkv == 1) a.kp_head = a.vp_head = 0;
    if (a.page_size == 1) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1) a.kp_page = a.vp_page = 0;
    const int64_t strides = a.q_token | a.q_head | a.out_token | a.out_head | a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head;
    KVC_REQUIRE((at & 15) == 0 && (strides & 7) == 0, "kvc_paged_attn: rows must start on 16 bytes");
    KVC_REQUIRE(a.kp_row >= 0 && a.kp_head >= 0 && a.vp_row >= 0 && a.vp_head >= 0 && a.kp_page >= 0 && a.vp_page >= 0 && a.kp_row * (a.page_size - 1) + a.kp_head * (a.Hkv - 1) < (1ll << 31) &&
                    a.vp_row * (a.page_size - 1) + a.vp_head * (a.Hkv - 1) < (1ll << 31), "kvc_paged_attn: a page spans more than 2^31 elements");
    KVC_REQUIRE(a.workspace && (reinterpret_cast<uintptr_t>(a.workspace) & 15) == 0, "kvc_paged_attn: the workspace must be 16-byte aligned");
    if (a.workspace_bytes < kvc_paged_attn_workspace(a.B, a.Hq, a.Hkv, a.D)) {
        kvc_set_error("kvc_paged_attn: the workspace must hold what kvc_paged_attn_workspace says");
        return KVC_ERR_CAPACITY;
    }
    const kvc_rows q = kvc_make_rows(a.q, a.D, rows, a.q_token, a.Hq, a.q_head), out = kvc_make_rows(a.out, a.D, rows, a.out_token, a.Hq, a.out_head);
    KVC_REQUIRE(out.apart, "kvc_paged_attn: rows of the output overlap");
    KVC_REQUIRE(kvc_rows_equal(q, out) || !kvc_rows_overlap(q, out), "kvc_paged_attn: the output overlaps the queries and is not them");
    Params p;
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
    cudaStream_t s = kvc_cu(stream);
    p.v_less_k = reinterpret_cast<const uint8_t *>(a.vpages) - reinterpret_cast<const uint8_t *>(a.kpages);
    const bool same = a.kp_page == a.vp_page && a.kp_row == a.vp_row && a.kp_head == a.vp_head;
    return a.type == KVC_TYPE_FP16 ? choose<__half>(p, same, s) : choose<__nv_bfloat16>(p, same, s);
}

extern "C" int kvc_paged_attn(const kvc_paged_attn_args *args, kvc_stream_t stream) { return paged_attn(args, nullptr, 0, stream); }
extern "C" int kvc_paged_attn_rows(const kvc_paged_attn_args *args, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(starts, "kvc_paged_attn_rows: null pointer");
    return paged_attn(args, starts, rows, stream);
}
