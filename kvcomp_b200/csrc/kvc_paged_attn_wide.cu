// Attention of one new token per request over pages, results in 32 bits: for calls with prefixes, which join them with others.  (kvc_paged_attn.cuh has the kernel.)
#include "kvc_paged_attn.cuh"

namespace kvc_paged {
namespace {

// (as for results of 16 bits; pools of different strides take the kernel that asks for both, those of the same strides too where two KV heads are not read together)
template <typename T, int D, int STAGES, int CTAS, int WIDE_STAGES, int WIDE_CTAS>
int choose_heads(Params &p, bool same, cudaStream_t s) {
    if (p.group > 8) return launch_kernel<T, D, 2, 1, false, WIDE_STAGES, WIDE_CTAS, true, WIDE_RESULTS>(p, s);
    if constexpr (D < 128) {
        if (same && p.per_head == 1 && p.a.Hkv % 2 == 0 && p.a.kp_head < p.a.kp_row) return launch_kernel<T, D, 1, 2, true, STAGES, CTAS, true, WIDE_RESULTS>(p, s);
    }
    return launch_kernel<T, D, 1, 1, false, STAGES, CTAS, true, WIDE_RESULTS>(p, s);
}

template <typename T>
int choose(Params &p, bool same, cudaStream_t s) {
    switch (p.a.D) {
        case 64: return choose_heads<T, 64, 3, 4, 4, 3>(p, same, s);
        case 96: return choose_heads<T, 96, 3, 3, 4, 2>(p, same, s);
        default: return choose_heads<T, 128, 2, 3, 3, 2>(p, same, s);
    }
}

}  // namespace

int launch_wide(Params &p, cudaStream_t s) {
    const kvc_paged_attn_args &a = p.a;
    const bool same = a.kp_page == a.vp_page && a.kp_row == a.vp_row && a.kp_head == a.vp_head;
    return a.type == KVC_TYPE_FP16 ? choose<__half>(p, same, s) : choose<__nv_bfloat16>(p, same, s);
}

}  // namespace kvc_paged
