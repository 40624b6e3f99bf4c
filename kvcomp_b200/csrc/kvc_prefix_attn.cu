// Attention of one new token per request where requests continue a common prefix: the prefix is read once for all that follow it.
//
// out = sum_t w_t v_t / sum_t w_t with w_t = exp(scaling q . k_t - m), over the tokens of the prefix and the request's own ones.  The sums of any parts of the tokens are kept with their
// maxima and joined.  Three kernels: prefixes, times all queries that follow them; the requests' own tokens (the kernel of calls without prefixes, with results of 32 bits); the joining.
//
// What bounds the first: of n requests with g query heads on a KV head, n g rows meet every key and value of the prefix, 4 n g D operations for 4 D bytes: HBM up to some 250 rows, the tensor
// cores and the exponentials beyond.  mma.sync (what the second kernel uses, at 8 rows) gives a quarter of that; so here tcgen05: 128 rows by 128 tokens, the scores in tensor
// memory, the weights in 16 bits in their place as the second product's operand, the sums there too.  Two sets of 128 rows take turns: while the exponentials of one are made the other's
// products run.  Columns of more than 128 rows use both sets with the same tokens; columns of fewer give them every other tile.
//
// Work is cut into tiles of 128 tokens of a column (a prefix's KV head and up to 256 of its followers' rows), all tiles of all columns in one row; each CTA, one on an SM, takes an
// equal, contiguous share, found from the lengths in the kernel.  What a CTA finds for a column goes to the workspace; the third kernel joins the parts, in the order of the
// shares, so that results do not depend on timing.
//
// Keys and values come by 16-byte asynchronous copies (pages end anywhere, any strides) into a ring in shared memory, in the 128-byte swizzled layout that the products read: keys
// channel by channel, values as they lie (token by token: the product's second operand turned).  Rounding: a weight has two pieces of fp16
// (times 2^7) or bf16, as in the kernel of calls without prefixes, and the second product is made with both: who follows a prefix has results as exact as who holds the same tokens.  Sums of weights
// are taken before that; everything joined is 32 bits and the result is rounded once.  (Of one piece: 58.5 us for the first call below, and 1.35 times the error against 64 bits.)
//
// Measured, device times of one B200: 64 requests of 32 heads behind 16384 tokens of 8 KV heads (256 rows a KV head), 1 to 500 own tokens each, 64 us: prefix 41, own tokens 23 (some of it beside the
// prefix's end), joining 10.  Of the 41, 5 pass before the first tile's scores (lengths, pages, first bytes, one behind the other) and 4 with 19 MB of parts; a tile's exponentials alone take 2048
// cycles, its products half as many again.  8 times 16 requests of 40 heads behind 8000 tokens of 10 (64 rows a KV head) 135 us: prefix 70 (280 MB, 4 TB/s), own tokens 66, joining 10.  4 requests of 32 heads
// behind 777 tokens 15.4 us: three kernels' starts.  (Joined where the own tokens' columns end, without a third kernel, 2 to 22 us more: few threads read many parts then, and hold what others
// need meanwhile.)
#include <math_constants.h>
#include <string.h>

#include <algorithm>

#include "kvc_paged_attn.cuh"

namespace {

using kvc_paged::Params, kvc_paged::set_params, kvc_paged::launch_wide, kvc_paged::counter_bytes, kvc_paged::places, kvc_paged::group_of, kvc_paged::part_floats, kvc_paged::columns_of, kvc_paged::check_rows, kvc_paged::check_results;

constexpr int PREFIX_THREADS = 512, QUERY_LOADERS = 3, ROWS = 128, TOKENS = 128, ATOM = 16384;       // ATOM: 128 rows of 128 bytes
constexpr int MASKS = 16;
constexpr int MAX_REQUESTS = 16384;

// Places in a plan of B requests, in words: what is asked for together lies together.
__host__ __device__ constexpr int64_t plan_groups(int64_t) { return 4; }                   // groups [B][4]: first member, members (0 behind the last group), whose prefix it is, how long
__host__ __device__ constexpr int64_t plan_owners(int64_t B) { return 4 + 4 * B; }         // requests [B][2]: group (-1: none), place among its members
__host__ __device__ constexpr int64_t plan_order(int64_t B) { return 4 + 6 * B; }          // members, group by group [B]
__host__ __device__ constexpr int64_t plan_leader(int64_t B) { return 4 + 7 * B; }         // scratch: the first of those with the same prefix, their number [B] each
__host__ __device__ constexpr int64_t plan_count(int64_t B) { return 4 + 8 * B; }
__host__ __device__ constexpr int64_t plan_words(int64_t B) { return 4 + 9 * B; }          // (the first: groups)

// ---- the plan: requests with the same prefix become a group ---------------------------------------------------------

constexpr int FIND_THREADS = 256, SCAN_THREADS = 1024;

struct Wish { int parent, shared; };
__device__ __forceinline__ Wish wish_of(const kvc_prefix_plan_args &a, int b, int &flags) {
    Wish w = {a.parents[b], a.shared[b]};
    if (w.parent < 0) return {-1, 0};
    if (w.parent >= a.B || w.parent == b || w.shared < 0) { flags |= KVC_FLAG_BAD_LENGTH; return {-1, 0}; }
    return w;
}

// For each request the first with the same prefix, how many of these are before it and how many there are: all are looked at, which for 1024 requests takes a few us and is done when
// requests come, not for every step.
__global__ void __launch_bounds__(FIND_THREADS) prefix_find_kernel(const __grid_constant__ kvc_prefix_plan_args a) {
    __shared__ Wish wishes[FIND_THREADS];
    kvc_behind();
    const int B = (int)a.B, b = blockIdx.x * FIND_THREADS + threadIdx.x;
    int flags = 0, ignored = 0;
    const Wish mine = b < B ? wish_of(a, b, flags) : Wish{-1, 0};
    if (mine.parent >= 0 && a.parents[mine.parent] >= 0) flags |= KVC_FLAG_BAD_LENGTH;     // who is followed follows no one
    int leader = -1, rank = 0, count = 0;
    for (int first = 0; first < B; first += FIND_THREADS) {
        __syncthreads();
        wishes[threadIdx.x] = first + (int)threadIdx.x < B ? wish_of(a, first + threadIdx.x, ignored) : Wish{-1, 0};
        __syncthreads();
        const int n = min(FIND_THREADS, B - first);
        for (int i = 0; i < n; i++) {
            if (wishes[i].parent != mine.parent || wishes[i].shared != mine.shared) continue;
            if (leader < 0) leader = first + i;
            rank += first + i < b;
            count++;
        }
    }
    if (b < B) {
        a.plan[plan_leader(B) + b] = mine.parent < 0 ? -1 : leader;
        a.plan[plan_owners(B) + 2 * b + 1] = rank;
        a.plan[plan_count(B) + b] = count;
    }
    raise_flag(a.status, flags);
}

__global__ void __launch_bounds__(SCAN_THREADS) prefix_scan_kernel(const __grid_constant__ kvc_prefix_plan_args a) {
    __shared__ int2 warps[SCAN_THREADS / 32];
    __shared__ int2 before_s;
    kvc_behind();
    const int B = (int)a.B, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int ignored = 0;
    if (threadIdx.x == 0) before_s = make_int2(0, 0);
    __syncthreads();                                        // (of no requests the loop, and its barriers, are left out)
    for (int b0 = 0; b0 < B; b0 += SCAN_THREADS) {
        const int b = b0 + threadIdx.x;
        const bool leads = b < B && a.plan[plan_leader(B) + b] == b;
        const int count = leads ? a.plan[plan_count(B) + b] : 0;
        int2 sum = make_int2(leads, count);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
            if (lane >= o) { sum.x += x; sum.y += y; }
        }
        if (lane == 31) warps[warp] = sum;
        __syncthreads();
        int2 before = before_s;
        for (int w = 0; w < warp; w++) { before.x += warps[w].x; before.y += warps[w].y; }
        const int group = before.x + sum.x - leads, first = before.y + sum.y - count;
        if (leads) {
            const Wish w = wish_of(a, b, ignored);
            int32_t *const to = a.plan + plan_groups(B) + 4 * group;
            to[0] = first; to[1] = count; to[2] = w.parent; to[3] = w.shared;
            a.plan[plan_owners(B) + 2 * b] = group;
        }
        __syncthreads();
        if (threadIdx.x == SCAN_THREADS - 1) before_s = make_int2(before.x + sum.x, before.y + sum.y);
        __syncthreads();
    }
    const int groups = before_s.x;
    if (threadIdx.x == 0) a.plan[0] = groups;
    for (int i = 4 * groups + threadIdx.x; i < 4 * B; i += SCAN_THREADS) a.plan[plan_groups(B) + i] = 0;
    for (int b = threadIdx.x; b < B; b += SCAN_THREADS) {
        const int leader = a.plan[plan_leader(B) + b];
        if (leader < 0) { a.plan[plan_owners(B) + 2 * b] = -1; continue; }
        const int group = a.plan[plan_owners(B) + 2 * leader];               // (written by this CTA ahead of a barrier)
        if (leader != b) a.plan[plan_owners(B) + 2 * b] = group;
        a.plan[plan_order(B) + a.plan[plan_groups(B) + 4 * group] + a.plan[plan_owners(B) + 2 * b + 1]] = b;
    }
}

// ---- the attention --------------------------------------------------------------------------------------------------

struct Prefix {
    kvc_paged_attn_args a;
    const int32_t *plan, *starts;                           // starts null: row b is request b's
    kvc_div page, group;                                    // divisors: page size, query heads of a KV head
    int g, rows, most_tokens, grid;                         // query heads of a KV head, rows of q, tokens of a table row, CTAs
    unsigned n_pages;
    int negative;
    float log2_scaling;
    int4 *items;                                            // (workspace) the groups' first tiles, tiles of a column, rows of a KV head, tiles of a share
    float *own, *own_lse;                                   // (workspace) results of the requests' own tokens [request][query head][D], logarithms of their sums
    float *sums;                                            // (workspace) of places of D floats
    float2 *maxima;                                         // maximum and sum of weights of a place
};

// Places: of column parts that begin with the column [request][head][2]; behind them of those that begin with a CTA's share [CTA][256].
__device__ __forceinline__ long long place_of(const Prefix &p, int b, int h, int i) { return (b * p.a.Hq + h) * 2 + i; }
__device__ __forceinline__ long long cta_place(const Prefix &p, int cta, int i) { return p.a.B * p.a.Hq * 2 + (long long)cta * 256 + i; }

__device__ __forceinline__ int row_at(const Prefix &p, int b) { return p.starts ? min(max(p.starts[b], 0), p.rows) : b; }
__device__ __forceinline__ int member_at(const Prefix &p, int i) { return min(max(p.plan[plan_order(p.a.B) + i], 0), (int)p.a.B - 1); }
// the row of a request's token, -1: it has none, or more than one
__device__ __forceinline__ int row_of(const Prefix &p, int b) {
    if (!p.starts) return b;
    const int row = row_at(p, b);
    return row_at(p, b + 1) - row == 1 ? row : -1;
}
__device__ __forceinline__ int length_of(const Prefix &p, int b) { return min(max(p.a.lengths[b], 0), p.most_tokens); }

struct Item { int table, first, rows, len, tiles, parts; bool cut; };       // whose pages, the first member in the order, rows of a KV head, tokens, tiles of a column, columns of a KV head; fewer tokens than are shared
__device__ __forceinline__ Item item_of(const Prefix &p, int i) {
    Item r;
    const int B = (int)p.a.B;
    const int4 group = *reinterpret_cast<const int4 *>(p.plan + plan_groups(B) + 4 * i);
    r.first = min(max(group.x, 0), B);                      // (kept inside the arrays whatever the plan holds, as lengths are)
    r.rows = min(max(group.y, 0), B - r.first) * p.g;
    r.table = min(max(group.z, 0), B - 1);
    r.len = r.rows == 0 ? 0 : min(max(group.w, 0), length_of(p, r.table));
    r.cut = r.rows > 0 && r.len < group.w;
    r.tiles = (r.len + TOKENS - 1) / TOKENS;
    r.parts = (r.rows + 2 * ROWS - 1) / (2 * ROWS);
    return r;
}

// A CTA's way through its share, column by column; the same for all its warps.
struct Walk {
    int item, column, tile, left, in_part;                  // the first tile of the column's part in this share, tiles of the share that are left, of the part
    int tiles_before, jobs;                                 // of the share, before the part
    int k_head, part;
    Item it;
    bool wide;                                              // more than one set's rows: a tile is two jobs, else one, of the sets in turn
};
__device__ __forceinline__ void begin_part(Walk &w) {
    w.k_head = w.column / w.it.parts;
    w.part = w.column - w.k_head * w.it.parts;
    w.wide = w.it.rows - w.part * 2 * ROWS > ROWS;
    w.in_part = min(w.it.tiles - w.tile, w.left);
}
__device__ __forceinline__ void next_part(const Prefix &p, Walk &w, int groups) {
    w.jobs += w.wide ? 2 * w.in_part : w.in_part;
    w.tiles_before += w.in_part;
    if ((w.left -= w.in_part) == 0) return;
    w.tile = 0;
    if (++w.column == w.it.parts * (int)p.a.Hkv) {
        w.column = 0;
        do {
            if (++w.item >= groups) { w.left = 0; return; }     // (lengths that changed meanwhile)
            w.it = item_of(p, w.item);
        } while (w.it.tiles == 0);
    }
    begin_part(w);
}

// ---- what the hardware is asked for
__device__ __forceinline__ uint32_t shared_at(const void *v) { return (uint32_t)__cvta_generic_to_shared(v); }
__device__ __forceinline__ void bar_init(uint64_t *bar, int count) { asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(shared_at(bar)), "r"(count)); }
__device__ __forceinline__ void bar_arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(shared_at(bar)) : "memory"); }
__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(shared_at(bar)), "r"(parity) : "memory");
    return done;
}
__device__ __forceinline__ bool bar_done(uint64_t *bar, uint32_t parity) {                // (try_wait may take some 10000 cycles to say no)
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(shared_at(bar)), "r"(parity) : "memory");
    return done;
}
// Waits up to about a second; what runs out is said in *failed, and nothing waits any more then.
__device__ __forceinline__ void bar_wait(uint64_t *bar, uint32_t parity, volatile int *failed) {
    if (bar_try(bar, parity)) return;
    const long long until = clock64() + (1ll << 31);
    while (!bar_try(bar, parity)) {
        if (*failed) return;
        if (clock64() > until) { *failed = 1; return; }
    }
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void seen_by_products() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// One lane of the warp asks for products and what follows them; all lanes come along, so that what these take is the warp's (uniform registers) and not put together by a lane for every one:
// 32 products and commits of a tile took 6000 cycles of one lane alone.
__device__ __forceinline__ uint32_t one_lane() {
    uint32_t is;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(is));
    return is;
}
__device__ __forceinline__ void commit_to(uint32_t one, uint64_t *bar) {
    asm volatile("{ .reg .pred e; setp.ne.u32 e, %1, 0; @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(shared_at(bar)), "r"(one) : "memory");
}
// operands in shared memory, 128-byte swizzle: of 1024-byte pieces (8 rows) that follow one another; `other` bytes to the next 64 channels where rows are not what is summed over.  Sixteen
// bytes further: one more.
__device__ __forceinline__ uint64_t operand_at(uint32_t at, uint32_t other) {
    return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(other >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void product(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{ .reg .pred p, e; setp.ne.u32 p, %4, 0; setp.ne.u32 e, %5, 0; @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add), "r"(one) : "memory");
}
__device__ __forceinline__ void product_of_weights(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{ .reg .pred p, e; setp.ne.u32 p, %4, 0; setp.ne.u32 e, %5, 0; @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(kind), "r"((uint32_t)add), "r"(one) : "memory");
}
#define KVC_32(X) X(0), X(1), X(2), X(3), X(4), X(5), X(6), X(7), X(8), X(9), X(10), X(11), X(12), X(13), X(14), X(15), X(16), X(17), X(18), X(19), X(20), X(21), X(22), X(23), X(24), X(25), X(26), X(27), X(28), X(29), X(30), X(31)
__device__ __forceinline__ void load32(uint32_t *r, uint32_t at) {
#define KVC_OUT(i) "=r"(r[i])
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
                 "%28, %29, %30, %31}, [%32];" : KVC_32(KVC_OUT) : "r"(at));
#undef KVC_OUT
}
__device__ __forceinline__ void store32(uint32_t at, const uint32_t *r) {
#define KVC_IN(i) "r"(r[i])
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
                 "%28, %29, %30, %31};" ::KVC_32(KVC_IN), "r"(at) : "memory");
#undef KVC_IN
}
__device__ __forceinline__ void loads_wait(uint32_t *r) {    // (nothing of r is used before)
#define KVC_BOTH(i) "+r"(r[i])
    asm volatile("tcgen05.wait::ld.sync.aligned;" : KVC_32(KVC_BOTH)::"memory");
#undef KVC_BOTH
}
__device__ __forceinline__ void stores_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// two at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x; }" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ void store_sector(void *to, const uint32_t *r) {               // 32 bytes, of a lane's own row: a whole sector
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Rows 32 i .. 32 i + 31 of a tile, by a warp: `from` is the lane's own row, mask says which there are (the others become zeros).  between() is called when a quarter is on its way.
template <typename T, int D, typename F> __device__ __forceinline__ void copy_rows(uint32_t to, int i, const T *from, uint32_t mask, int lane, F between) {
    constexpr int SIDE = D == 96 ? 4 : D / 8 > 16 ? 16 : D / 8;                           // lanes of a row
#pragma unroll 1
    for (int k0 = 0; k0 < SIDE; k0 += 4) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int j = (k0 + k) * (32 / SIDE) + lane / SIDE, r = 32 * i + j;
            const T *row = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), j));
#pragma unroll
            for (int c0 = 0; c0 < D / 8; c0 += SIDE) {
                const int c = c0 + lane % SIDE;
                copy16(to + (c >> 3) * ATOM + r * 128 + ((c & 7) ^ (r & 7)) * 16, row + c * 8, mask >> j & 1);
            }
        }
        if (k0 == 0) between();
    }
}

template <typename T> struct Weight;
template <> struct Weight<__half> { static constexpr float LIFT = 7.0f; static constexpr uint32_t KIND = 0; };
template <> struct Weight<__nv_bfloat16> { static constexpr float LIFT = 0.0f; static constexpr uint32_t KIND = 1; };
constexpr float SLACK = 8.0f;                               // the maximum that weights go by is put up when it is 2^8 too low: the sums are touched once or twice a column, not every tile

template <int D> struct Shape {
    static constexpr int ATOMS = (D + 63) / 64, UNIT = ATOMS * ATOM, RING = ATOMS == 1 ? 10 : 5;      // a tile of keys or values; how many lie in the ring
    static constexpr size_t SHARED = (size_t)(2 + RING) * UNIT + 1024;
};

template <typename T, int D>
__global__ void __launch_bounds__(PREFIX_THREADS, 1) prefix_attn_kernel(const __grid_constant__ Prefix p) {
    constexpr int UNIT = Shape<D>::UNIT, RING = Shape<D>::RING;
    constexpr float LIFT = Weight<T>::LIFT;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[RING], empty[RING], scores_there[2], weights_there[2], sums_there[2], queries_there[2], queries_free[2], over;
    __shared__ uint32_t masks[MASKS][4], tensor_s;
    __shared__ int failed_s, warp_sums[PREFIX_THREADS / 32], start_item, start_rest;
    __shared__ Item start_it;
    const kvc_paged_attn_args &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = (int)a.B;
    volatile int *failed = &failed_s;
    const uint32_t base = (shared_at(raw) + 1023) & ~1023u, ring = base + 2 * UNIT;

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_at(&tensor_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        for (int i = 0; i < RING; i++) { bar_init(full + i, 4); bar_init(empty + i, 1); }
        for (int i = 0; i < 2; i++) { bar_init(scores_there + i, 1); bar_init(weights_there + i, 4); bar_init(sums_there + i, 1); bar_init(queries_there + i, 4); bar_init(queries_free + i, 1); }
        bar_init(&over, 1);
        failed_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }

    // ---- this CTA's share
    kvc_behind();                                           // (from here on the kernel of the requests' own tokens, which reads nothing of this one's, may begin where there is room)
    const int groups = min(max(p.plan[0], 0), B), looked_at = max(groups, min(B, PREFIX_THREADS));       // (those behind the last have no members: the first are looked at before their number is there)
    int flags = 0, total = 0;
    Item it = {};
    auto scan = [&](int i0, int &tiles) {                   // (first tile of item i0 + tid, its tiles; `total` grows)
        it.tiles = it.parts = 0;
        it.cut = false;
        if (i0 + tid < B) it = item_of(p, i0 + tid);
        if (it.cut) flags |= KVC_FLAG_BAD_LENGTH;
        tiles = it.tiles * it.parts * (int)a.Hkv;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        __syncthreads();
        if (lane == 31) warp_sums[warp] = sum;
        __syncthreads();
        int before = total;
        for (int w = 0; w < PREFIX_THREADS / 32; w++) {
            if (w < warp) before += warp_sums[w];
            total += warp_sums[w];
        }
        return before + sum - tiles;
    };
    int tiles = 0, first = 0;
    for (int i0 = 0; i0 < looked_at; i0 += PREFIX_THREADS) first = scan(i0, tiles);
    const int all = total, size = max(1, (all + p.grid - 1) / p.grid), r0 = (int)min((long long)all, (long long)size * blockIdx.x), r1 = r0 + min(size, all - r0);
    if (r0 < r1 || blockIdx.x == 0) {                       // (of more groups than threads the first CTA and those with work look twice)
        if (groups > PREFIX_THREADS) total = 0;
        for (int i0 = 0; i0 < groups; i0 += PREFIX_THREADS) {
            if (groups > PREFIX_THREADS) first = scan(i0, tiles);
            if (blockIdx.x == 0 && i0 + tid < groups) p.items[i0 + tid] = make_int4(first, it.tiles, it.rows, size);
            if (r0 >= first && r0 < first + tiles) { start_item = i0 + tid; start_rest = r0 - first; start_it = it; }
        }
    }
    if (blockIdx.x > 0) flags = 0;                          // (one says it)
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tensor = tensor_s;

    if (r0 < r1) {
        Walk w;
        w.left = r1 - r0;
        w.jobs = w.tiles_before = 0;
        w.item = start_item;
        w.it = start_it;
        w.column = start_rest / w.it.tiles;
        w.tile = start_rest - w.column * w.it.tiles;
        begin_part(w);

        if (warp < 8) {
            // ---- a set of rows: scores -> weights, and the sums' way out
            const int set = warp >> 2, r = tid & 127;
            const uint32_t lanes = (uint32_t)(warp & 3) << 21, scores = tensor + lanes + set * 128, sums = tensor + lanes + 256 + set * 128;
            const uint32_t lowest = p.negative ? 0x7f800000u : 0xff800000u;                // (before they are scaled)
            int phase = 0, parts = 0;                       // of this set's jobs, of its columns' parts
            for (; w.left > 0; next_part(p, w, groups)) {
                const int idx = (set - w.jobs) & 1, half = w.wide ? idx : 0, first_n = w.wide ? 0 : idx, step = w.wide ? 1 : 2;
                if (first_n >= w.in_part) continue;
                const int R = w.part * 2 * ROWS + half * ROWS + r;
                bool mine = R < w.it.rows;
                long long place = 0;
                if (mine) {
                    const int member = kvc_divide(R, p.group), h = w.k_head * p.g + R - member * p.g, b = member_at(p, w.it.first + member);
                    mine = row_of(p, b) >= 0;
                    place = w.tile == 0 ? place_of(p, b, h, first_n) : cta_place(p, blockIdx.x, (w.wide ? half : first_n) * ROWS + r);
                }
                const bool some = __any_sync(0xffffffffu, mine);
                float m = -CUDART_INF_F, l = 0.0f;
                for (int n = first_n; n < w.in_part; n += step) {
                    bar_wait(scores_there + set, phase, failed);
                    after_sync();
                    if (some) {
                        const uint32_t *const mask = masks[(w.tiles_before + n) % MASKS];
                        if ((mask[0] & mask[1] & mask[2] & mask[3]) != 0xffffffffu) {      // tokens that are none (a column's last tile, bad pages): their scores become the lowest
#pragma unroll 1
                            for (int c = 0; c < 4; c++) {
                                uint32_t x[32];
                                load32(x, scores + 32 * c);
                                loads_wait(x);
                                const uint32_t on = mask[c];
#pragma unroll
                                for (int i = 0; i < 32; i++) x[i] = on >> i & 1 ? x[i] : lowest;
                                store32(scores + 32 * c, x);
                            }
                            stores_wait();
                        }
                        // Twice over the scores, 32 at a time (all 128 at once would not leave registers enough): their maximum, then the weights.  Loops of two steps: all four in a row are
                        // more instructions than are at hand when the sets come by (64 requests behind 16384 tokens 48 us, so 40).
                        uint32_t x[32], y[32];
                        float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
                        auto highest = [&](const uint32_t *v) {
                            if (p.negative) {
#pragma unroll
                                for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], -__uint_as_float(v[i]));
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i++) top[i & 3] = max3(top[i & 3], __uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                            }
                        };
                        load32(x, scores);
#pragma unroll 1
                        for (int c = 0; c < 2; c++) {
                            loads_wait(x);
                            load32(y, scores + 64 * c + 32);
                            highest(x);
                            loads_wait(y);
                            load32(x, scores + (c == 0 ? 64 : 0));       // (and the first again)
                            highest(y);
                        }
                        const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * fabsf(p.log2_scaling);
                        const bool up = high > m + SLACK || (m == -CUDART_INF_F && high > m);
                        if (__any_sync(0xffffffffu, up)) {
                            const float now = up ? high : m, f = up ? exp2_approx(m - now) : 1.0f;
                            m = now;
                            l *= f;
                            if (n != first_n) {             // (the sums are there: what was asked for behind them is)
                                loads_wait(x);
#pragma unroll 1
                                for (int c = 0; c < D / 32; c++) {
                                    load32(y, sums + 32 * c);
                                    loads_wait(y);
#pragma unroll
                                    for (int i = 0; i < 32; i++) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                                    store32(sums + 32 * c, y);
                                }
                            }
                        }
                        const float less = LIFT - (m == -CUDART_INF_F ? 0.0f : m);
                        const float2 scale2 = make_float2(p.log2_scaling, p.log2_scaling), less2 = make_float2(less, less);
                        float2 sum[2] = {};
                        auto weigh = [&](const uint32_t *v, uint32_t to) {       // (weights take the scores' own place: 16 columns, and 16 of what is left of them)
                            uint32_t weights[32];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float2 e = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scale2, less2);
                                const float2 f = make_float2(exp2_approx(e.x), exp2_approx(e.y));
                                sum[i & 1] = add2(sum[i & 1], f);
                                weights[i] = pack(f.x, f.y, T());
                                const float2 g = unpack(weights[i], T()), r = add2(f, make_float2(-g.x, -g.y));
                                weights[16 + i] = pack(r.x, r.y, T());
                            }
                            store32(to, weights);
                        };
#pragma unroll 1
                        for (int c = 0; c < 2; c++) {
                            loads_wait(x);
                            load32(y, scores + 64 * c + 32);
                            weigh(x, scores + 64 * c);
                            loads_wait(y);
                            if (c == 0) load32(x, scores + 64);
                            weigh(y, scores + 64 * c + 32);
                        }
                        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        stores_wait();
                    }
                    before_sync();
                    __syncwarp();
                    if (lane == 0) bar_arrive(weights_there + set);
                    phase ^= 1;
                }
                bar_wait(sums_there + set, parts, failed);
                parts ^= 1;
                after_sync();
                if (some) {
                    uint32_t o[2][32];
                    load32(o[0], sums);
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        loads_wait(o[c & 1]);
                        if (c + 1 < D / 32) load32(o[(c + 1) & 1], sums + 32 * (c + 1));
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < 4; i++) store_sector(p.sums + place * D + 32 * c + 8 * i, o[c & 1] + 8 * i);
                        }
                    }
                    if (mine) __stcg(p.maxima + place, make_float2(m - LIFT, l));          // (weights were 2^LIFT times what the maximum says)
                }
                before_sync();
            }
        } else {
            if (warp == 8) {
                // ---- the products
                constexpr uint32_t KIND = 1u << 4 | Weight<T>::KIND << 7 | Weight<T>::KIND << 10 | (uint32_t)(ROWS >> 4) << 24;
                constexpr uint32_t SCORES = KIND | (uint32_t)(TOKENS >> 3) << 17, VALUES = KIND | 1u << 16 | (uint32_t)(D >> 3) << 17;
                auto all_lanes = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
                const uint32_t one = one_lane(), t_at = (uint32_t)all_lanes((int)tensor);
                const uint64_t queries = operand_at(base, 16), keys = operand_at(ring, 16), values = operand_at(ring, ATOM);
                int slot = 0, round = 0;                    // of the ring: the next unit's place, and how often it has been through (its last bit)
                auto next_unit = [&]() { if (++slot == RING) { slot = 0; round ^= 1; } };
                int phases = 0;                             // a bit for each set: its jobs, the lowest two; the next two: its queries
                // Of each set the job that waits for its second product, and where its values lie.  A set's scores may be written again when its weights have been read: its next first product
                // is asked for right behind its second one, and products are made in order.
                struct { int slot, round; bool there, first, last, ends; } late[2] = {};
                auto second = [&](int set) {
                    const auto &job = late[set];
                    if (!job.there) return;
                    bar_wait(full + job.slot, job.round, failed);
                    bar_wait(weights_there + set, phases >> set & 1, failed);
                    phases ^= 1 << set;
                    after_sync();
                    const uint64_t b = values + (uint32_t)job.slot * (UNIT / 16);
                    const uint32_t d = t_at + 256 + set * 128, a_at = t_at + set * 128;
#pragma unroll
                    for (int k = 0; k < TOKENS / 16; k++) {         // (of 32 tokens the weights, 16 columns, then what is left of them)
                        product_of_weights(one, d, a_at + k / 2 * 32 + k % 2 * 8, b + k * (2048 / 16), VALUES, k > 0 || !job.first);
                        product_of_weights(one, d, a_at + k / 2 * 32 + k % 2 * 8 + 16, b + k * (2048 / 16), VALUES, true);
                    }
                    if (job.last) commit_to(one, empty + job.slot);
                    if (job.ends) commit_to(one, sums_there + set);
                };
                int odd = 0, pending = -1;                  // the next job's set; the set whose values are still to come
                for (; all_lanes(w.left) > 0; next_part(p, w, groups)) {
                    const int in_part = all_lanes(w.in_part);
                    const bool wide = all_lanes(w.wide);
                    for (int n = 0; n < in_part; n++) {
                        const bool begins = wide ? n == 0 : n < 2, ends = wide ? n == in_part - 1 : n + 2 >= in_part;
                        const int k_slot = slot;
                        bar_wait(full + slot, round, failed);
                        next_unit();
                        if (pending >= 0) {                 // the values of the tile before come behind this one's keys
                            if (pending) late[1].slot = slot, late[1].round = round;
                            else late[0].slot = slot, late[0].round = round;
                            next_unit();
                        }
                        const int v_slot = slot, v_round = round;       // (wide)
                        if (wide) next_unit();
                        auto job = [&](int set, bool last) {
                            second(set);
                            if (begins) {
                                bar_wait(queries_there + set, phases >> (2 + set) & 1, failed);
                                phases ^= 4 << set;
                            }
                            after_sync();
                            const uint64_t q_at = queries + set * (UNIT / 16), k_at = keys + (uint32_t)k_slot * (UNIT / 16);
                            const uint32_t d = t_at + set * 128;
#pragma unroll
                            for (int k = 0; k < D / 16; k++) product(one, d, q_at + ((k >> 2) * ATOM + (k & 3) * 32) / 16, k_at + ((k >> 2) * ATOM + (k & 3) * 32) / 16, SCORES, k > 0);
                            commit_to(one, scores_there + set);
                            if (ends) commit_to(one, queries_free + set);
                            if (last) commit_to(one, empty + k_slot);
                            late[set] = {v_slot, v_round, true, begins, last, ends};
                            odd ^= 1;
                        };
                        for (int j = 0; j < (wide ? 2 : 1); j++) {
                            const bool last = !wide || j == 1;
                            if (odd) job(1, last);
                            else job(0, last);
                        }
                        pending = wide ? -1 : odd ^ 1;
                    }
                }
                if (pending >= 0) {
                    if (pending) late[1].slot = slot, late[1].round = round;
                    else late[0].slot = slot, late[0].round = round;
                }
                if (odd) { second(1); second(0); }
                else { second(0); second(1); }
                commit_to(one, &over);                      // all products are done before anything is given back
                bar_wait(&over, 0, failed);
                __syncwarp();
            } else if (warp < 13) {
                // ---- the copies of keys and values: each of four warps has 32 rows of every tile, whose pages it asks for a tile ahead
                const int i = warp - 9;
                constexpr int ON_THE_WAY = RING > 5 ? 4 : 2;               // units whose copies are on their way while the next ones are asked for
                uint64_t *signals[ON_THE_WAY] = {};         // where to say that they are there, the oldest first
                auto say = [&](uint64_t *bar) {
                    seen_by_products();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar);
                };
                auto drain = [&]() {
                    copies_wait<0>();
#pragma unroll
                    for (int k = 0; k < ON_THE_WAY; k++) {
                        if (signals[k]) say(signals[k]);
                        signals[k] = nullptr;
                    }
                };
                auto oldest = [&]() {                       // (called when the first copies of the next unit are on their way)
                    if (!signals[0]) return;
                    copies_wait<ON_THE_WAY - 1>();
                    say(signals[0]);
                };
                // Units of the ring in the order of their use: a tile's keys, and its values behind the next tile's keys (narrow: the next job's first product runs before them) or behind
                // its own (wide).
                int slot = 0, round = 1;                    // the next unit's place; the bit to wait for there (1: the first time round there is nothing to wait for)
                auto send = [&](bool values, int page, uint32_t mask, int t, int k_head) {
                    if (!__all_sync(0xffffffffu, bar_done(empty + slot, round))) {
                        drain();                            // (what is waited for may need what this warp has copied)
                        bar_wait(empty + slot, round, failed);
                        __syncwarp();
                    }
                    const T *from = reinterpret_cast<const T *>(values ? a.vpages : a.kpages);
                    const int row = t - kvc_divide(t, p.page) * (int)a.page_size;
                    if (mask >> lane & 1) from += values ? page * a.vp_page + row * a.vp_row + k_head * a.vp_head : page * a.kp_page + row * a.kp_row + k_head * a.kp_head;
                    copy_rows<T, D>(ring + slot * UNIT, i, from, mask, lane, oldest);
                    copies_commit();
#pragma unroll
                    for (int k = 0; k + 1 < ON_THE_WAY; k++) signals[k] = signals[k + 1];
                    signals[ON_THE_WAY - 1] = full + slot;
                    if (++slot == RING) { slot = 0; round ^= 1; }
                };
                int tile_n = 0, late_page = 0, late_t = 0, late_head = 0;
                uint32_t late_mask = 0;
                bool late = false;                          // values that are still to come
                for (; w.left > 0; next_part(p, w, groups)) {
                    const int32_t *const pages = a.table + w.it.table * a.table_stride;
                    int t = w.tile * TOKENS + 32 * i + lane, page = t < w.it.len ? pages[kvc_divide(t, p.page)] : -1;
                    for (int n = 0; n < w.in_part; n++, tile_n++, t += TOKENS) {
                        const int behind = t + TOKENS, next = n + 1 < w.in_part && behind < w.it.len ? pages[kvc_divide(behind, p.page)] : -1;
                        const bool good = (unsigned)page < p.n_pages;
                        if (!good && t < w.it.len) flags |= KVC_FLAG_BAD_PAGE;
                        const uint32_t mask = __ballot_sync(0xffffffffu, good);
                        if (lane == 0) masks[tile_n % MASKS][i] = mask;
                        send(false, page, mask, t, w.k_head);
                        if (late) send(true, late_page, late_mask, late_t, late_head);
                        late = !w.wide;
                        if (w.wide) send(true, page, mask, t, w.k_head);
                        late_page = page; late_mask = mask; late_t = t; late_head = w.k_head;
                        page = next;
                    }
                }
                if (late) send(true, late_page, late_mask, late_t, late_head);
                drain();
            } else {
                // ---- the copies of queries: the columns' rows, 32 at a time, by three warps in turn
                int block = warp - 13, loads0 = 0, loads1 = 0;      // times the sets' queries were loaded
                for (; w.left > 0; next_part(p, w, groups)) {
                    const int sets = w.wide || w.in_part > 1 ? 2 : 1;           // (narrow: both sets have the same rows)
                    for (; block < 4 * sets; block += QUERY_LOADERS) {
                        const int j = block >> 2, i = block & 3, set = (w.jobs + j) & 1, loads = set ? loads1 : loads0;
                        const int R = w.part * 2 * ROWS + (w.wide ? j * ROWS : 0) + 32 * i + lane, member = kvc_divide(R, p.group);
                        int row = R < w.it.rows ? member_at(p, w.it.first + member) : -1;
                        if (row >= 0) row = row_of(p, row);
                        if (loads > 0) bar_wait(queries_free + set, (loads - 1) & 1, failed);
                        __syncwarp();
                        const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
                        if (mask) copy_rows<T, D>(base + set * UNIT, i, reinterpret_cast<const T *>(a.q) + (row >= 0 ? (long long)row * a.q_token + (w.k_head * p.g + R - member * p.g) * a.q_head : 0), mask, lane, []() {});
                        copies_commit();
                        copies_wait<0>();
                        seen_by_products();
                        __syncwarp();
                        if (lane == 0) bar_arrive(queries_there + set);
                    }
                    block -= 4 * sets;
                    if (sets == 2) loads0++, loads1++;
                    else if (w.jobs & 1) loads1++;
                    else loads0++;
                }
            }
        }
    }
    if (flags && a.status) atomicOr(a.status, flags);
    before_sync();
    __syncthreads();
    after_sync();
    if (tid == 0 && failed_s && a.status) atomicOr(a.status, KVC_FLAG_WAIT_TIMEOUT);
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tensor));
}

// ---- the parts of a row's sums are joined ---------------------------------------------------------------------------

// Writes the result v of query head h of request b, four channels a lane, some of which came out as no numbers although the sum of weights is one, by the definition (as calls without prefixes have
// it): a value of +inf or -inf that counts makes the result that, both, or one that is no number itself, or one of weight 0 (a score of -inf), none.  For each four channels that hold such a one the
// warp reads these of the prefix's and the request's own values again, a token a lane, until nothing can change.  In line and small: behind a call, or with eight tokens a lane, all calls took 5 to
// 7 us more (64 requests behind 16384 tokens).  One infinity among these 364 us.
template <typename T, int D> __device__ __forceinline__ void write_with_infinities(const Prefix &p, int b, int row, int h, int owner, int groups, float4 v) {
    constexpr uint32_t INFINITE = Weight<T>::KIND ? 0x7f80u : 0x7c00u;
    const kvc_paged_attn_args &a = p.a;
    const int lane = threadIdx.x & 31, hk = kvc_divide(h, p.group);
    Item item = {};
    if (owner >= 0 && owner < groups) item = item_of(p, owner);
    const T *const q = reinterpret_cast<const T *>(a.q) + row * a.q_token + h * a.q_head;
    const uint32_t none = lane >= D / 4 ? 0 : (v.x != v.x) | (v.y != v.y) << 1 | (v.z != v.z) << 2 | (v.w != v.w) << 3;
    uint32_t sign = 0;                                      // of each channel: 1 +inf, 2 -inf, 3 none
#pragma unroll 1
    for (uint32_t pieces = __ballot_sync(0xffffffffu, none != 0); pieces; pieces &= pieces - 1) {
        const int piece = __ffs(pieces) - 1;
        uint32_t seen = 0;
#pragma unroll 1
        for (int part = 0; part < 2; part++) {
            const int32_t *const pages = a.table + (part ? b : item.table) * a.table_stride;
            const int len = part ? length_of(p, b) : item.len;
#pragma unroll 1
            for (int t0 = 0; t0 < len && seen != 0xff; t0 += 32) {
                const int t = t0 + lane, page = t < len ? pages[kvc_divide(t, p.page)] : -1, r = t - kvc_divide(t, p.page) * (int)a.page_size;
                uint32_t here = 0;
                if ((unsigned)page < p.n_pages) {
                    const uint2 x = *reinterpret_cast<const uint2 *>(reinterpret_cast<const T *>(a.vpages) + page * a.vp_page + r * a.vp_row + hk * a.vp_head + 4 * piece);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint32_t y = (c < 2 ? x.x : x.y) >> c % 2 * 16 & 0xffff;
                        if ((y & INFINITE) == INFINITE) here |= ((y & 0x7fff) != INFINITE ? 3u : y & 0x8000 ? 2u : 1u) << 2 * c;
                    }
                    if (here) {
                        const T *const key = reinterpret_cast<const T *>(a.kpages) + page * a.kp_page + r * a.kp_row + hk * a.kp_head;
                        float score = 0.0f;
#pragma unroll 1
                        for (int c = 0; c < D; c++) score += (float)q[c] * (float)key[c];
                        if ((p.negative ? -score : score) == -CUDART_INF_F) here |= (here >> 1 & 0x55) | (here << 1 & 0xaa);      // the weight is 0
                    }
                }
                seen |= __reduce_or_sync(0xffffffffu, here);
            }
        }
        if (lane == piece) sign = seen;
    }
    float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t of = sign >> 2 * c & 3;
        if (none >> c & 1) r[c] = of == 1 ? CUDART_INF_F : of == 2 ? -CUDART_INF_F : CUDART_NAN_F;
    }
    if (lane < D / 4) *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + row * a.out_token + h * a.out_head + lane * 4) = make_uint2(pack(r[0], r[1], T()), pack(r[2], r[3], T()));
}

// A warp for a row's head, or (TEAM 4) four, which take the parts in turn, their sums joined in the warps' order.  Few rows have columns of many parts, eight at a time in flight: the call for
// 2 x 3 requests of 14 heads behind 31212 tokens, 148 parts a head, takes 28 us with four warps and 34 with one; 64 requests of 32 heads behind 16384, 18 parts a head, 65.4 with four and 63 with
// one.
template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(128) prefix_join_kernel(const __grid_constant__ Prefix p) {
    kvc_behind();
    const kvc_paged_attn_args &a = p.a;
    const int lane = threadIdx.x & 31, B = (int)a.B, warp = threadIdx.x >> 5;
    const int of_request = TEAM == 1 ? (int)(a.Hq + 3) / 4 : (int)a.Hq, b = blockIdx.x / of_request, h = (blockIdx.x - b * of_request) * (4 / TEAM) + (TEAM == 1 ? warp : 0);
    __shared__ float4 sums_s[TEAM == 1 ? 1 : TEAM][32];
    __shared__ float2 maxima_s[TEAM];
    if (h >= a.Hq) return;
    const bool on = lane < D / 4;
    auto nothing = [&](int row) {
        if (on) *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + row * a.out_token + h * a.out_head + lane * 4) = make_uint2(0, 0);
        if (lane == 0 && a.lse) a.lse[row * a.Hq + h] = -CUDART_INF_F;
    };
    if (b == B) {                                           // rows behind the last
        for (int row = row_at(p, B); row < p.rows; row++) nothing(row);
        return;
    }
    // (what does not wait for anything else is asked for together: the request's row and group, the result of its own tokens and the logarithm of their weights' sum)
    const int2 owner = *reinterpret_cast<const int2 *>(p.plan + plan_owners(B) + 2 * b);
    const int row = row_at(p, b), behind = p.starts ? row_at(p, b + 1) : b + 1, groups = min(p.plan[0], B);
    const float own = TEAM == 1 || warp == 0 ? __ldcg(p.own_lse + b * a.Hq + h) : -CUDART_INF_F;
    float4 v = on ? __ldcg(reinterpret_cast<const float4 *>(p.own + (b * a.Hq + h) * D) + lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int4 it = p.items[min(max(owner.x, 0), B - 1)];
    if (behind - row != 1) {
        for (int i = row; i < behind; i++) nothing(i);
        return;
    }
    const int k_head = kvc_divide(h, p.group);
    float top = own * 1.4426950408889634f, sum = own == -CUDART_INF_F ? 0.0f : 1.0f;
    if (own == -CUDART_INF_F) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float2 ml, float4 x) {
        const float now = fmaxf(top, ml.x), less = now == -CUDART_INF_F ? 0.0f : now, f = exp2_approx(top - less), g = exp2_approx(ml.x - less);
        sum = sum * f + ml.y * g;
        // (what nothing was added to may hold anything)
        v.x = v.x * f + x.x * g; v.y = v.y * f + x.y * g; v.z = v.z * f + x.z * g; v.w = v.w * f + x.w * g;
        top = now;
    };
    constexpr int AT_ONCE = 8;
    int count = 0;                                          // the parts
    if (owner.x >= 0 && owner.x < groups && it.y > 0) {
        const int size = max(it.w, 1), parts = (it.z + 2 * ROWS - 1) / (2 * ROWS);
        const int R = min(max(owner.y, 0), it.z / p.g - 1) * p.g + h - k_head * p.g, part = R / (2 * ROWS), in_part = R - part * 2 * ROWS;
        const bool wide = it.z - part * 2 * ROWS > ROWS;
        const int from = it.x + (k_head * parts + part) * it.y, to = from + it.y;
        // a column's parts: each in a CTA's share, of narrow columns two (every other tile) where it has more than one
        const int cta0 = from / size, cta1 = (to - 1) / size, each = wide ? 1 : 2;
        count = (cta1 - cta0 + 1) * each;
        for (int k0 = TEAM == 1 ? 0 : warp * AT_ONCE; k0 < count; k0 += TEAM * AT_ONCE) {
            float2 ml[AT_ONCE];
            float4 x[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const int cta = cta0 + (k0 + k) / each, which = (k0 + k) % each;
                const int there = min(to, (cta + 1) * size) - max(from, cta * size);
                ml[k] = make_float2(-CUDART_INF_F, 0.0f);
                x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (cta <= cta1 && which < there) {
                    const long long place = cta == cta0 ? place_of(p, b, h, which) : cta_place(p, cta, wide ? in_part : which * ROWS + in_part);
                    ml[k] = __ldcg(p.maxima + place);
                    if (on) x[k] = __ldcg(reinterpret_cast<const float4 *>(p.sums + place * D) + lane);
                }
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++)
                if (ml[k].x != -CUDART_INF_F || ml[k].y != 0.0f) add(ml[k], x[k]);
        }
    }
    if (TEAM > 1 && count > AT_ONCE) {                            // (the count is the CTA's)
        if (lane == 0) maxima_s[warp % TEAM] = make_float2(top, sum);
        sums_s[warp % TEAM][lane] = v;
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 1; w < TEAM; w++)
            if (maxima_s[w].x != -CUDART_INF_F || maxima_s[w].y != 0.0f) add(maxima_s[w], sums_s[w][lane]);
    }
    if (TEAM > 1 && warp > 0) return;
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    if (lane == 0 && a.lse) a.lse[row * a.Hq + h] = sum == 0.0f ? -CUDART_INF_F : (top + log2f(sum)) * 0.69314718055994531f;
    const float any = v.x + v.y + v.z + v.w;
    if (__any_sync(0xffffffffu, any != any && sum == sum)) {
        write_with_infinities<T, D>(p, b, row, h, owner.x, groups, v);
        return;
    }
    if (on) *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + row * a.out_token + h * a.out_head + lane * 4) = make_uint2(pack(v.x, v.y, T()), pack(v.z, v.w, T()));
}

template <typename T, int D>
int launch(Prefix &p, Params &own, cudaStream_t s) {
    static kvc_launch_slot slot;
    int occ = 0;
    if (int rc = kvc_prepare(slot, reinterpret_cast<const void *>(prefix_attn_kernel<T, D>), PREFIX_THREADS, Shape<D>::SHARED, &occ)) return rc;
    KVC_REQUIRE(occ > 0, "kvc_paged_attn_shared: the kernel does not fit this device");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3(PREFIX_THREADS);
    cfg.dynamicSmemBytes = Shape<D>::SHARED;
    cfg.stream = s;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    KVC_CUDA_OK(cudaLaunchKernelEx(&cfg, prefix_attn_kernel<T, D>, (const Prefix)p));
    if (int rc = launch_wide(own, s)) return rc;
    // (four warps a head as long as that makes no more CTAs than SMs)
    if ((p.a.B + 1) * p.a.Hq <= kvc_sm_count()) return kvc_launch_early(prefix_join_kernel<T, D, 4>, (unsigned)((p.a.B + 1) * p.a.Hq), 128, s, p);
    return kvc_launch_early(prefix_join_kernel<T, D, 1>, (unsigned)((p.a.B + 1) * ((p.a.Hq + 3) / 4)), 128, s, p);
}

int64_t rounded(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t prefix_places(int64_t B, int64_t Hq) { return 2 * B * Hq + 256ll * kvc_sm_count(); }
int64_t own_bytes(int64_t Hq, int64_t Hkv, int64_t D) { return rounded(counter_bytes() + places(D) * part_floats(group_of(Hq, Hkv, D), D) * 4); }      // of the kernel for own tokens

}  // namespace

extern "C" int64_t kvc_prefix_plan_words(int64_t B) { return B < 0 ? 0 : plan_words(B); }

extern "C" int kvc_prefix_plan(const kvc_prefix_plan_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_prefix_plan: null pointer");
    kvc_prefix_plan_args a;
    memcpy(&a, args, sizeof(a));
    KVC_REQUIRE(a.B >= 0 && a.B <= MAX_REQUESTS, "kvc_prefix_plan: %lld requests, %d at most", (long long)a.B, MAX_REQUESTS);
    KVC_REQUIRE((reinterpret_cast<uintptr_t>(a.plan) & 15) == 0, "kvc_prefix_plan: the plan must be 16-byte aligned");
    KVC_REQUIRE(a.plan && (a.B == 0 || (a.parents && a.shared)), "kvc_prefix_plan: null pointer");
    cudaStream_t s = kvc_cu(stream);
    if (a.B > 0)
        if (int rc = kvc_launch_early(prefix_find_kernel, (unsigned)((a.B + FIND_THREADS - 1) / FIND_THREADS), FIND_THREADS, s, a)) return rc;
    return kvc_launch_early(prefix_scan_kernel, 1, SCAN_THREADS, s, a);
}

extern "C" int64_t kvc_paged_attn_shared_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    if (B < 0 || Hkv <= 0 || Hq < Hkv || D <= 0) return 0;
    return own_bytes(Hq, Hkv, D) + rounded(16 * B) + rounded(4 * B * Hq * (D + 1)) + prefix_places(B, Hq) * (4 * D + 8);
}

extern "C" int kvc_paged_attn_shared(const kvc_paged_attn_args *args, const int32_t *plan, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(args && plan, "kvc_paged_attn_shared: null pointer");
    KVC_REQUIRE((reinterpret_cast<uintptr_t>(plan) & 15) == 0, "kvc_paged_attn_shared: the plan must be 16-byte aligned");
    Prefix p;
    memcpy(&p.a, args, sizeof(p.a));
    kvc_paged_attn_args &a = p.a;
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_paged_attn_shared: unknown type %d", a.type);
    KVC_REQUIRE(a.D == 64 || a.D == 96 || a.D == 128, "kvc_paged_attn_shared: heads of 64, 96 or 128 channels, got %lld", (long long)a.D);
    KVC_REQUIRE(a.B >= 0 && a.B <= MAX_REQUESTS && a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0 && a.Hq < 65536, "kvc_paged_attn_shared: %lld query heads over %lld", (long long)a.Hq, (long long)a.Hkv);
    KVC_REQUIRE(a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages >= 0 && a.n_pages < (1ll << 31) && a.table_width >= 0, "kvc_paged_attn_shared: bad sizes");
    KVC_REQUIRE(a.window == 0, "kvc_paged_attn_shared: no window (it would end inside the prefix)");
    KVC_REQUIRE(a.table_width * a.page_size < (1ll << 31) - 256, "kvc_paged_attn_shared: a table row holds %lld tokens, lengths have 32 bits", (long long)(a.table_width * a.page_size));
    if (!starts) rows = a.B;
    KVC_REQUIRE(rows >= 0 && rows < (1 << 24) && (a.B > 0 || rows == 0), "kvc_paged_attn_shared: %lld rows of %lld requests", (long long)rows, (long long)a.B);
    if (rows == 0) return KVC_OK;
    KVC_REQUIRE(a.q && a.out && a.lengths && (a.table || a.table_width == 0) && ((a.kpages && a.vpages) || a.n_pages == 0), "kvc_paged_attn_shared: null pointer");
    const int64_t g = a.Hq / a.Hkv, most_tiles = (a.table_width * a.page_size + TOKENS - 1) / TOKENS;
    KVC_REQUIRE(a.Hkv * (2 * a.B + a.B * g / (2 * ROWS)) < (1ll << 30) / std::max<int64_t>(most_tiles, 1), "kvc_paged_attn_shared: requests, KV heads and table rows of more than 2^30 tiles");
    KVC_REQUIRE(a.B * columns_of(a.Hq, a.Hkv, a.D) * ((a.table_width * a.page_size + 31) / 32) < (1ll << 31) - (1 << 20), "kvc_paged_attn_shared: requests, KV heads and table rows of more than 2^31 tiles");
    if (int rc = check_rows(a, rows, 8, "kvc_paged_attn_shared")) return rc;              // (the kernel for own tokens goes by them too)
    KVC_REQUIRE(a.workspace && (reinterpret_cast<uintptr_t>(a.workspace) & 31) == 0, "kvc_paged_attn_shared: the workspace must be 32-byte aligned");         // (sums are written by whole sectors)
    if (a.workspace_bytes < kvc_paged_attn_shared_workspace(a.B, a.Hq, a.Hkv, a.D)) {
        kvc_set_error("kvc_paged_attn_shared: the workspace must hold what kvc_paged_attn_shared_workspace says");
        return KVC_ERR_CAPACITY;
    }
    if (int rc = check_results(a, rows, "kvc_paged_attn_shared")) return rc;
    p.plan = plan;
    p.starts = starts;
    p.page = kvc_make_div((uint32_t)a.page_size);
    p.group = kvc_make_div((uint32_t)g);
    p.g = (int)g;
    p.rows = (int)rows;
    p.most_tokens = (int)(a.table_width * a.page_size);
    p.grid = kvc_sm_count();
    p.n_pages = (unsigned)a.n_pages;
    p.negative = a.scaling < 0.0f;
    p.log2_scaling = std::max(fabsf(a.scaling) * 1.4426950408889634f, 1e-37f) * (p.negative ? -1.0f : 1.0f);      // (0 times the infinite score of a token that is left out is none)
    uint8_t *at_ws = reinterpret_cast<uint8_t *>(a.workspace) + own_bytes(a.Hq, a.Hkv, a.D);
    p.items = reinterpret_cast<int4 *>(at_ws);
    at_ws += rounded(16 * a.B);
    p.own = reinterpret_cast<float *>(at_ws);
    p.own_lse = p.own + a.B * a.Hq * a.D;
    at_ws += rounded(4 * a.B * a.Hq * (a.D + 1));
    p.sums = reinterpret_cast<float *>(at_ws);
    p.maxima = reinterpret_cast<float2 *>(p.sums + prefix_places(a.B, a.Hq) * a.D);
    Params own = {};
    set_params(own, a, starts, rows);
    own.wide = p.own;
    own.a.lse = p.own_lse;
    cudaStream_t s = kvc_cu(stream);
    const bool fp16 = a.type == KVC_TYPE_FP16;
    if (a.D == 64) return fp16 ? launch<__half, 64>(p, own, s) : launch<__nv_bfloat16, 64>(p, own, s);
    if (a.D == 96) return fp16 ? launch<__half, 96>(p, own, s) : launch<__nv_bfloat16, 96>(p, own, s);
    return fp16 ? launch<__half, 128>(p, own, s) : launch<__nv_bfloat16, 128>(p, own, s);
}
