// Attention of one new token per request over pages of 8-bit codes: which kernel.  (kvc_paged_attn.cuh has the kernel.)
#include "kvc_paged_attn.cuh"

namespace kvc_paged {
namespace {

// As for rows of 16 bits (a stage has twice the tokens and the same bytes, and their scales); 96 channels with a stage less, which three CTAs need to fit an SM.  Rows of 64 and 96 channels of two KV
// heads are read together, as there (8 x 4096 tokens of 32 heads of 96 channels in int8 56 us, one by one 69; 16 x 16384 of 8 heads of 64 in e4m3 with a query head each 76 and 77.6, with eight 80.4 and 79.2).
template <typename T, int D, int STAGES, int CTAS, int WIDE_STAGES, int WIDE_CTAS, int KIND>
int choose_heads(Params &p, cudaStream_t s) {
    if constexpr (WIDE_STAGES > 0) {
        if (p.group > 8) return launch<T, D, 2, 1, true, WIDE_STAGES, WIDE_CTAS, KIND>(p, s);
    }
    if constexpr (D < 128) {
        if (p.per_head == 1 && p.a.Hkv % 2 == 0 && p.a.kp_head < p.a.kp_row) return launch<T, D, 1, 2, true, STAGES, CTAS, KIND>(p, s);
    }
    return launch<T, D, 1, 1, true, STAGES, CTAS, KIND>(p, s);
}

template <typename T, int KIND>
int choose(Params &p, cudaStream_t s) {
    switch (p.a.D) {
        case 64: return choose_heads<T, 64, 3, 4, 4, 3, KIND>(p, s);
        case 96: return choose_heads<T, 96, 2, 3, 3, 2, KIND>(p, s);
        case 128: return choose_heads<T, 128, 2, 3, 3, 2, KIND>(p, s);
        default: return choose_heads<T, 256, 3, 1, 0, 0, KIND>(p, s);
    }
}

}  // namespace

int launch_codes(Params &p, cudaStream_t s) {
    if (p.a.type == KVC_TYPE_FP16) return p.s.codes == KVC_CODES_INT8 ? choose<__half, KVC_CODES_INT8>(p, s) : choose<__half, KVC_CODES_E4M3>(p, s);
    return p.s.codes == KVC_CODES_INT8 ? choose<__nv_bfloat16, KVC_CODES_INT8>(p, s) : choose<__nv_bfloat16, KVC_CODES_E4M3>(p, s);
}

}  // namespace kvc_paged
