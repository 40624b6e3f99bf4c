// Attention of one new token per request over pages: which kernel, and the C entries.  (kvc_paged_attn.cuh has the kernel.)
#include "kvc_paged_attn.cuh"

namespace {

using namespace kvc_paged;

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

}  // namespace

extern "C" int64_t kvc_paged_attn_cleared(void) { return counter_bytes(); }
extern "C" int64_t kvc_paged_attn_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    if (B < 0 || Hkv <= 0 || Hq < Hkv || D <= 0) return 0;
    return counter_bytes() + places(D) * part_floats(group_of(Hq, Hkv, D), D) * 4;
}

// starts null: a row for each request; scales null: pools of the queries' type
static int paged_attn(const kvc_paged_attn_args *args, const kvc_scales *scales, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_paged_attn: null pointer");
    kvc_paged_attn_args a;
    kvc_scales c = {};
    memcpy(&a, args, sizeof(a));
    if (scales) memcpy(&c, scales, sizeof(c));
    KVC_REQUIRE(!scales || c.codes == KVC_CODES_INT8 || c.codes == KVC_CODES_E4M3, "kvc_paged_attn_codes: unknown codes %d", c.codes);
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
    if (int rc = check_rows(a, rows, scales ? 16 : 8, "kvc_paged_attn")) return rc;
    KVC_REQUIRE(a.workspace && (reinterpret_cast<uintptr_t>(a.workspace) & 15) == 0, "kvc_paged_attn: the workspace must be 16-byte aligned");
    if (a.workspace_bytes < kvc_paged_attn_workspace(a.B, a.Hq, a.Hkv, a.D)) {
        kvc_set_error("kvc_paged_attn: the workspace must hold what kvc_paged_attn_workspace says");
        return KVC_ERR_CAPACITY;
    }
    if (int rc = check_results(a, rows, "kvc_paged_attn")) return rc;
    Params p = {};
    set_params(p, a, starts, rows);
    cudaStream_t s = kvc_cu(stream);
    const bool same = a.kp_page == a.vp_page && a.kp_row == a.vp_row && a.kp_head == a.vp_head;
    if (scales) {
        if (a.Hkv == 1) c.k_head = c.v_head = 0;
        if (a.n_pages <= 1) c.k_page = c.v_page = 0;
        KVC_REQUIRE((c.k && c.v) || a.n_pages == 0, "kvc_paged_attn_codes: null pointer");
        KVC_REQUIRE(same && c.k_page == c.v_page && c.k_head == c.v_head, "kvc_paged_attn_codes: keys and values, and their scales, must have the same strides");
        KVC_REQUIRE(((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 3) == 0, "kvc_paged_attn_codes: scales must start on 4 bytes");
        p.s = c;
        return launch_codes(p, s);
    }
    return a.type == KVC_TYPE_FP16 ? choose<__half>(p, same, s) : choose<__nv_bfloat16>(p, same, s);
}

extern "C" int kvc_paged_attn(const kvc_paged_attn_args *args, kvc_stream_t stream) { return paged_attn(args, nullptr, nullptr, 0, stream); }
extern "C" int kvc_paged_attn_rows(const kvc_paged_attn_args *args, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(starts, "kvc_paged_attn_rows: null pointer");
    return paged_attn(args, nullptr, starts, rows, stream);
}
extern "C" int kvc_paged_attn_codes(const kvc_paged_attn_args *args, const kvc_scales *scales, const int32_t *starts, int64_t rows, kvc_stream_t stream) {
    KVC_REQUIRE(scales, "kvc_paged_attn_codes: null pointer");
    return paged_attn(args, scales, starts, rows, stream);
}
