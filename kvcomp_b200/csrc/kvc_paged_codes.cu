// Paged caches whose tokens are held in 8 bits: rows are coded as they go to their slots, and read back.
//
// A row (a token's channels of a KV head, keys after their rotation) has one scale s in 32 bits.  int8: s = max |x| / 127, codes x / s to the nearest whole number, ties to even.
// e4m3: s = the least power of two with max |x| / s <= 448, codes x / s to the nearest e4m3: a power of two costs a floating code nothing, and the quotient is exact.  No scale is
// below 2^-100, so that its inverse and its products are numbers.  A row that holds an infinity or no number has no scale: NaN, and all of it reads back so.
//
// Every value is read once and written once: HBM for a prompt, latency for a step, as for rows of 16 bits; the codes are a part of the instructions only where that does not show.
#include <cuda_fp8.h>
#include <math_constants.h>
#include <string.h>

#include <algorithm>

#include "kvc_paged.cuh"

namespace {

struct CodesParams {
    kvc_rotary_args a;
    kvc_scales s;
    kvc_div page;
    long long slots;                                        // of the pool
    int lanes, units, tokens;                               // lanes of a row (a power of two), those that have channels; tokens of a CTA
    Part parts[3];
    int ctas;                                               // for these tokens: one for every few heads
    kvc_div by_ctas;
};

constexpr int CODES_THREADS = 128, CODES_CTAS = 5, CHUNK = 4;
constexpr float LEAST_SCALE = 7.888609052210118e-31f;       // 2^-100

// bits of |x|, so that what is no number is the largest
__device__ __forceinline__ uint32_t size_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a row by its largest size, and one over it.
template <int KIND> __device__ __forceinline__ float scale_of(uint32_t top, float &inverse) {
    float s;
    if (KIND == KVC_CODES_INT8) {
        // top / 127 rounded: a product with the rounded reciprocal, and its remainder, exact, times that (Markstein, Computation of elementary functions on the IBM RISC System/6000
        // processor, 1990)
        constexpr float LESS = 1.0f / 127.0f;
        const float t = __uint_as_float(top), q = t * LESS;
        s = fmaxf(fmaf(fmaf(-127.0f, q, t), LESS, q), LEAST_SCALE);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s));
    } else {                                                // top = m 2^e, 448 = 1.75 2^8: e - 8, one more where m is above 1.75
        const int e = max((int)((top + 0x1fffffu) >> 23) - 8, 127 - 100);
        s = __uint_as_float((uint32_t)e << 23);
        inverse = __uint_as_float((uint32_t)(254 - e) << 23);
    }
    if (top >= 0x7f800000u) s = CUDART_NAN_F;
    return s;
}

// two at a time, each rounded
__device__ __forceinline__ float2 mul2(float2 a, float b) {
    float2 r;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %4}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float b, float2 c) {
    float2 r;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %4}; mov.b64 z, {%5, %6}; fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x; }" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b), "f"(c.x), "f"(c.y));
    return r;
}
// the largest size of three; no number if one is none
__device__ __forceinline__ float largest(float a, float b, float c) {
    float r;
    asm("{ .reg .f32 x, y; abs.f32 x, %2; abs.f32 y, %3; max.NaN.f32 %0, %1, x, y; }" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Codes of 4 N values of a row, packed.  int8: x times one over s (off by 2^-23 of it) is off by 127 1.5 2^-23 of a step at most, so the whole number next to it is right unless it lies that near the border
// of two.  There the remainder x - q s says: it is a multiple of s's last bit and no larger than s, hence exact.
template <int KIND, int N> __device__ __forceinline__ void codes_of(const float *x, float s, float inverse, uint32_t *packed) {
    if (KIND == KVC_CODES_INT8) {
        constexpr float WHOLE = 12582912.0f;                // 1.5 2^23: a sum's last bits are a whole number's
        float2 w[2 * N];
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * N; i++) {
            const float2 t = mul2(make_float2(x[2 * i], x[2 * i + 1]), inverse);
            w[i] = add2(t, make_float2(WHOLE, WHOLE));
            const float2 q = add2(w[i], make_float2(-WHOLE, -WHOLE)), rest = add2(t, make_float2(-q.x, -q.y));
            far = largest(far, rest.x, rest.y);
        }
        if (far > 0.4999f) {
#pragma unroll
            for (int i = 0; i < 4 * N; i++) {
                float &c = i & 1 ? w[i / 2].y : w[i / 2].x;
                const float q = c - WHOLE, r = fmaf(-q, s, x[i]), d = 2.0f * fabsf(r);
                if (d > s || (d == s && (__float_as_uint(c) & 1))) c += r > 0.0f ? 1.0f : -1.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            packed[i] = __byte_perm(__byte_perm(__float_as_uint(w[2 * i].x), __float_as_uint(w[2 * i].y), 0x0040), __byte_perm(__float_as_uint(w[2 * i + 1].x), __float_as_uint(w[2 * i + 1].y), 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float2 a = mul2(make_float2(x[4 * i], x[4 * i + 1]), inverse), b = mul2(make_float2(x[4 * i + 2], x[4 * i + 3]), inverse);
            packed[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16;
        }
    }
}

// A pair y0, y1 rotated in 32 bits is off by NEAR times |y0| + |y1| at most (the sum of its products' sizes is their length, and that no more than this): 2.5 2^-24 of a product by cos or sin (their
// argument's, their series' and their own rounding), three more for the factor, a product and the sum, one for the limits themselves.  e4m3 keys are those of a rotation without any error: where
// both limits have the same code that is the key's, and the few others (one of some 15000; without it some keys in a million get the code beside theirs, and one of hundreds where a pair's products
// cancel) are rotated in 64 bits.
constexpr float NEAR = 7.0f / 16777216.0f;
__device__ __forceinline__ uint32_t e4m3_of(float2 v) { return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3); }
// Codes of four such values and the sizes |y0| + |y1| of their pairs; far: NEAR over the scale.  Returns where those of the limits differ.
__device__ __forceinline__ uint32_t codes_within(const float *x, float s0, float s1, float s2, float s3, float inverse, float far, uint32_t &packed) {
    const float2 a = mul2(make_float2(x[0], x[1]), inverse), b = mul2(make_float2(x[2], x[3]), inverse);
    packed = e4m3_of(fma2(make_float2(s0, s1), -far, a)) | e4m3_of(fma2(make_float2(s2, s3), -far, b)) << 16;
    return packed ^ (e4m3_of(fma2(make_float2(s0, s1), far, a)) | e4m3_of(fma2(make_float2(s2, s3), far, b)) << 16);
}
// A value rotated in 64 bits, cut to 24, the last one 1 where something was cut off: it rounds to fewer as the value itself does, and is above a number of fewer bits where the value is.
__device__ __noinline__ float rotated_closely(double position, double frequency, float factor, float f0, float f1, bool second) {
    double turns = position * (frequency * TURNS_OF_RADIANS), c, s;
    turns -= rint(turns);
    sincospi(2.0 * turns, &s, &c);
    const double exact = (second ? f1 * c + f0 * s : f0 * c - f1 * s) * factor;
    const float cut = __double2float_rz(exact);
    return (double)cut == exact ? cut : __uint_as_float(__float_as_uint(cut) | 1);
}
// which bytes are not 0: a bit for each
__device__ __forceinline__ uint32_t bits_of(uint32_t bytes) { return ((__vcmpne4(bytes, 0) & 0x01010101u) * 0x10204080u) >> 28; }
// The codes of those of a thread's 16 values whose bit of `which` is set; turns: they are rotated.
template <typename T> __device__ __noinline__ void code_closely(uint32_t which, const T *src, uint8_t *dst, int apart, bool half, bool turns, double position, const double *frequencies, float factor, float inverse) {
#pragma unroll 1
    for (; which; which &= which - 1) {
        const int v = __ffs(which) - 1, k = half ? v & 7 : v >> 1, i0 = half ? k : 2 * k, i1 = half ? apart + k : 2 * k + 1;
        const bool second = half ? v >= 8 : v & 1;
        const float f0 = to_float(src[i0]), f1 = to_float(src[i1]);
        const float y = turns ? rotated_closely(position, frequencies[k], factor, f0, f1, second) : second ? f1 : f0;
        dst[second ? i1 : i0] = (uint8_t)__nv_cvt_float_to_fp8(y * inverse, __NV_SATFINITE, __NV_E4M3);
    }
}
// A row's largest value decides on its scale, 448 times a power of two being the border: 1.75 2^e.  It is off by 2 NEAR of itself (|y0| + |y1| is no more than twice it), 13 of its last bits there;
// next to the border one of the row's values may be above it and the largest in 32 bits not, or the other way round.
constexpr uint32_t OF_BORDER = 0x600000, LAST_BITS = 13;
__device__ __forceinline__ bool at_border(uint32_t top) { return ((top - OF_BORDER + LAST_BITS) & 0x7fffffu) <= 2 * LAST_BITS && top >> 23 >= 127 - 100 + 8; }       // (below, the scale is the least)
__device__ __forceinline__ uint32_t border_of(uint32_t top) { return (top & 0x7f800000u) | OF_BORDER; }
// whether one of a thread's 8 pairs has a value above it; turns: they are rotated
template <typename T> __device__ __noinline__ bool above_border(uint32_t border, const T *src, int apart, bool half, bool turns, double position, const double *frequencies, float factor) {
    bool above = false;
#pragma unroll 1
    for (int k = 0; k < 8; k++) {
        const float f0 = to_float(src[half ? k : 2 * k]), f1 = to_float(src[half ? apart + k : 2 * k + 1]);
        for (int second = 0; second < 2; second++) {
            float y = second ? f1 : f0;
            if (turns) {
                const float2 cs = turn_closely(position, frequencies[k] * TURNS_OF_RADIANS, factor);
                y = second ? f1 * cs.x + f0 * cs.y : f0 * cs.x - f1 * cs.y;
                if (size_of(y) + LAST_BITS >= border) y = rotated_closely(position, frequencies[k], factor, f0, f1, second);
            }
            above |= size_of(y) > border;
        }
    }
    return above;
}

// Where a token goes: its row in the pools (in codes) and its place among the scales; -1: nowhere
struct Place { long long k, v, ks, vs; };
__device__ __forceinline__ Place place_of(const CodesParams &p, int slot, int &flags) {
    const kvc_rotary_args &a = p.a;
    Place r = {-1, -1, 0, 0};
    if (slot < 0) return r;
    if (slot >= p.slots) { flags = KVC_FLAG_BAD_PAGE; return r; }
    const int page = kvc_divide(slot, p.page), row = slot - page * (int)a.page_size;
    r.k = page * a.kp_page + row * a.kp_row;
    r.v = page * a.vp_page + row * a.vp_row;
    r.ks = page * p.s.k_page + row;
    r.vs = page * p.s.v_page + row;
    return r;
}

// Heads of 16 n channels, rotated by multiples of 16, everything on 16 bytes.  As for rows of 16 bits a thread has a unit of 16 channels (8 pairs) of up to CHUNK heads of a token, whose
// angles it makes once; the lanes of a row are neighbours in a warp and find the row's largest value among them.  A CTA has the same few heads of several tokens, the next one the next
// heads of these: queries, which are bytes alone, and keys and values, which take instructions, run at the same time.
// Measured: 16384 tokens of 40 + 10 + 10 heads of 128 channels in int8 (463 MB) 94 us, 5.0 TB/s, one kind behind the other and one head at a time 147; four or six CTAs per SM (the latter
// spilling) 112, two heads of a thread 104, six 116.  e4m3 93, and 4099 tokens of 32 + 8 + 8 heads (93 MB) 21.
// (Where the second looks at values next to a border were made in the loop, 135 and 26.)
template <typename T, int KIND>
__global__ void __launch_bounds__(CODES_THREADS, CODES_CTAS) codes_rows_kernel(const __grid_constant__ CodesParams p) {
    kvc_behind();
    const kvc_rotary_args &a = p.a;
    const int of_tokens = kvc_divide((int)blockIdx.x, p.by_ctas), cta = (int)blockIdx.x - of_tokens * p.ctas;
    const int which = cta >= (int)p.parts[2].first ? 2 : (cta >= (int)p.parts[1].first ? 1 : 0);
    const Part &part = p.parts[which];
    const int turned = part.turned, u = (int)threadIdx.x & (p.lanes - 1), n = of_tokens * p.tokens + (int)threadIdx.x / p.lanes;        // (lanes: a power of two)
    if (n >= a.N) return;
    const bool on = u < p.units;
    const int h0 = (cta - (int)part.first) * part.chunk, heads = min(part.chunk, part.heads - h0);
    const bool half = a.layout == KVC_ROTARY_HALF && u < turned;
    const int c0 = half ? 8 * u : 16 * u, apart = half ? 8 * turned : 8;
    const T *src = reinterpret_cast<const T *>(part.src) + n * part.src_token + h0 * part.src_head + c0;
    // everything is asked for before anything is waited for: place, position and frequencies one after the other took half of the time
    const bool turns = u < turned;
    const int slot = which > 0 ? a.slots[n] : 0, position = turns ? a.positions[n] : 0;
    double2 f2[4];
#pragma unroll
    for (int k = 0; k < 4; k++) f2[k] = turns ? reinterpret_cast<const double2 *>(a.frequencies)[4 * u + k] : make_double2(0.0, 0.0);
    uint4 x[CHUNK][2];
#pragma unroll
    for (int j = 0; j < CHUNK; j++) {
        x[j][0] = x[j][1] = make_uint4(0, 0, 0, 0);
        if (on && j < heads) {
            x[j][0] = *reinterpret_cast<const uint4 *>(src);
            x[j][1] = *reinterpret_cast<const uint4 *>(src + apart);
        }
        src += part.src_head;
    }
    uint8_t *dst = nullptr;
    float *scale = nullptr;
    if (which > 0) {
        int flags = 0;
        const Place at = place_of(p, slot, flags);
        raise_flag(a.status, flags);
        if (at.k < 0) return;                               // (a token's lanes all go)
        dst = reinterpret_cast<uint8_t *>(part.dst) + (which == 1 ? at.k : at.v) + h0 * part.dst_head + c0;
        scale = which == 1 ? p.s.k + at.ks + h0 * p.s.k_head : p.s.v + at.vs + h0 * p.s.v_head;
    }
    float2 cs[8];
    if (turns) {
        const double at = a.inverse ? -(double)position : (double)position;
#pragma unroll
        for (int k = 0; k < 8; k++) cs[k] = turn_closely(at, (k & 1 ? f2[k / 2].y : f2[k / 2].x) * TURNS_OF_RADIANS, a.factor);
    }
    const unsigned row_lanes = (p.lanes == 32 ? 0xffffffffu : (1u << p.lanes) - 1) << (threadIdx.x & 31 & ~(p.lanes - 1));
    auto values_of = [&](const uint4 (&v)[2], float (&f)[16]) {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int m = 0; m < 8; m++) {
            const float2 g = unpack(w[m], T());
            f[2 * m] = g.x; f[2 * m + 1] = g.y;
        }
        if (!turns) return;
        // pairs: with halves a value of the first piece and its like of the second, else neighbours
        if (half) {
#pragma unroll
            for (int m = 0; m < 8; m++) {
                const float f0 = f[m], f1 = f[8 + m];
                f[m] = f0 * cs[m].x - f1 * cs[m].y;
                f[8 + m] = f1 * cs[m].x + f0 * cs[m].y;
            }
        } else {
#pragma unroll
            for (int m = 0; m < 8; m++) {
                const float f0 = f[2 * m], f1 = f[2 * m + 1];
                f[2 * m] = f0 * cs[m].x - f1 * cs[m].y;
                f[2 * m + 1] = f1 * cs[m].x + f0 * cs[m].y;
            }
        }
    };
    if (which == 0) {
        T *to = reinterpret_cast<T *>(part.dst) + n * part.dst_token + h0 * part.dst_head + c0;
#pragma unroll
        for (int j = 0; j < CHUNK; j++) {
            if (on && j < heads) {
                float f[16];
                values_of(x[j], f);
                *reinterpret_cast<uint4 *>(to) = make_uint4(pack(f[0], f[1], T()), pack(f[2], f[3], T()), pack(f[4], f[5], T()), pack(f[6], f[7], T()));
                *reinterpret_cast<uint4 *>(to + apart) = make_uint4(pack(f[8], f[9], T()), pack(f[10], f[11], T()), pack(f[12], f[13], T()), pack(f[14], f[15], T()));
            }
            to += part.dst_head;
        }
        return;
    }
    uint32_t exponents = 0, borders = 0, again[CHUNK / 2] = {};                             // (e4m3) of the heads' scales; rows at a border of scales; values at a border of codes
    const bool sure = !turns || (position == 0 && a.factor == 1.0f);                       // (what is not turned is as it was)
    // Two heads at a time: the way from a row's values to its scale is a chain, and two take little more than one.
#pragma unroll
    for (int j = 0; j < CHUNK; j += 2) {
        if (j >= heads) break;
        float f[2][16], top[2] = {0.0f, 0.0f}, s[2], inverse[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            values_of(x[j + i], f[i]);
#pragma unroll
            for (int m = 0; m < 8; m++) top[i] = largest(top[i], f[i][2 * m], f[i][2 * m + 1]);
        }
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            if (o >= p.lanes) break;
            const float other[2] = {__shfl_xor_sync(row_lanes, top[0], o), __shfl_xor_sync(row_lanes, top[1], o)};
            top[0] = larger(top[0], other[0]);
            top[1] = larger(top[1], other[1]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            s[i] = scale_of<KIND>(size_of(top[i]), inverse[i]);
            if (KIND == KVC_CODES_E4M3) {
                uint32_t e = __float_as_uint(s[i]) >> 23;
                if (part.turned > 0 && at_border(size_of(top[i]))) { borders |= 1u << (j + i); e = (size_of(top[i]) >> 23) - 8; }
                exponents |= (e & 0xff) << 8 * (j + i);
            }
            if (on && j + i < heads) {
                uint32_t c[4], unsure[4] = {};
                if (KIND == KVC_CODES_E4M3 && part.turned > 0) {
                    const float *const y = f[i], far = sure ? 0.0f : NEAR * inverse[i];
                    auto size = [&](int a, int b) { return fabsf(y[a]) + fabsf(y[b]); };
                    if (a.layout == KVC_ROTARY_HALF) {
#pragma unroll
                        for (int m = 0; m < 8; m += 4) {
                            const float s0 = size(m, m + 8), s1 = size(m + 1, m + 9), s2 = size(m + 2, m + 10), s3 = size(m + 3, m + 11);
                            unsure[m / 4] = codes_within(y + m, s0, s1, s2, s3, inverse[i], far, c[m / 4]);
                            unsure[m / 4 + 2] = codes_within(y + m + 8, s0, s1, s2, s3, inverse[i], far, c[m / 4 + 2]);
                        }
                    } else {
#pragma unroll
                        for (int m = 0; m < 16; m += 4) {
                            const float s0 = size(m, m + 1), s1 = size(m + 2, m + 3);
                            unsure[m / 4] = codes_within(y + m, s0, s0, s1, s1, inverse[i], far, c[m / 4]);
                        }
                    }
                } else {
                    codes_of<KIND, 2>(f[i], s[i], inverse[i], c);
                    codes_of<KIND, 2>(f[i] + 8, s[i], inverse[i], c + 2);
                }
                *reinterpret_cast<uint2 *>(dst) = make_uint2(c[0], c[1]);
                *reinterpret_cast<uint2 *>(dst + apart) = make_uint2(c[2], c[3]);
                if (u == 0) *scale = s[i];
                if (KIND == KVC_CODES_E4M3 && (unsure[0] | unsure[1] | unsure[2] | unsure[3]))
                    again[j / 2] |= (bits_of(unsure[0]) | bits_of(unsure[1]) << 4 | bits_of(unsure[2]) << 8 | bits_of(unsure[3]) << 12) << 16 * i;
            }
            dst += part.dst_head;
            scale += which == 1 ? p.s.k_head : p.s.v_head;
        }
    }
    // Second looks, few, behind all else: in the loop what they need would have to be kept beside what it does.
    if (KIND == KVC_CODES_E4M3 && which == 1 && (borders | again[0] | again[1])) {
        int ignored = 0;
        const Place at = place_of(p, slot, ignored);
        const double turned_by = a.inverse ? -(double)position : (double)position;
#pragma unroll 1
        for (int j = 0; j < heads; j++) {
            const T *const row = reinterpret_cast<const T *>(part.src) + n * part.src_token + (h0 + j) * part.src_head + c0;
            int e = exponents >> 8 * j & 0xff;
            uint32_t values = (j < 2 ? again[0] : again[1]) >> 16 * (j & 1) & 0xffff;
            if (borders >> j & 1) {                         // (a row's lanes all, or none) all of its codes go by what is found
                const uint32_t border = (uint32_t)(e + 8) << 23 | OF_BORDER;
                const bool above = on && above_border<T>(border, row, apart, half, turns, turned_by, a.frequencies + 8 * u, a.factor);
                e = max(e + (__any_sync(row_lanes, above) ? 1 : 0), 127 - 100);
                if (u == 0) p.s.k[at.ks + (h0 + j) * p.s.k_head] = __uint_as_float((uint32_t)e << 23);
                values = on ? 0xffff : 0;
            }
            if (values)
                code_closely<T>(values, row, reinterpret_cast<uint8_t *>(part.dst) + at.k + (h0 + j) * part.dst_head + c0, apart, half, turns, turned_by, a.frequencies + 8 * u, a.factor,
                                __uint_as_float((uint32_t)(254 - e) << 23));
        }
    }
}

// Any sizes and strides of what is read: a warp per row, a lane every 32nd channel, whose angle it makes for itself, and again for its code.  4099 tokens of 32 + 8 + 8 heads of 96 channels, 24 of
// them rotated, in e4m3 (70 MB) 71 us.
template <typename T, int KIND>
__global__ void __launch_bounds__(CODES_THREADS) codes_any_kernel(const __grid_constant__ CodesParams p) {
    kvc_behind();
    const kvc_rotary_args &a = p.a;
    const long long heads = a.Hq + 2 * a.Hkv, row = (long long)blockIdx.x * (CODES_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= a.N * heads) return;
    const int lane = threadIdx.x & 31, h = (int)(row % heads), D = (int)a.D, rotary = h < a.Hq + a.Hkv ? (int)a.rotary : 0;
    const long long n = row / heads;
    const T *x;
    T *y = nullptr;
    uint8_t *dst = nullptr;
    float *scale = nullptr;
    if (h < a.Hq) {
        x = reinterpret_cast<const T *>(a.q) + n * a.q_token + h * a.q_head;
        y = reinterpret_cast<T *>(a.q_out) + n * a.out_token + h * a.out_head;
    } else {
        const bool key = h < a.Hq + a.Hkv;
        const long long hk = h - a.Hq - (key ? 0 : a.Hkv);
        int flags = 0;
        const Place at = place_of(p, a.slots[n], flags);
        if (lane == 0) raise_flag(a.status, flags);
        if (at.k < 0) return;
        x = key ? reinterpret_cast<const T *>(a.k) + n * a.k_token + hk * a.k_head : reinterpret_cast<const T *>(a.v) + n * a.v_token + hk * a.v_head;
        dst = key ? reinterpret_cast<uint8_t *>(a.kpages) + at.k + hk * a.kp_head : reinterpret_cast<uint8_t *>(a.vpages) + at.v + hk * a.vp_head;
        scale = key ? p.s.k + at.ks + hk * p.s.k_head : p.s.v + at.vs + hk * p.s.v_head;
    }
    const double position = rotary == 0 ? 0.0 : a.inverse ? -(double)a.positions[n] : (double)a.positions[n];
    auto pair_of = [&](int i, int &other, bool &second) {   // a rotated channel's pair
        const int half = rotary / 2;
        second = a.layout == KVC_ROTARY_HALF ? i >= half : i & 1;
        other = a.layout == KVC_ROTARY_HALF ? (second ? i - half : i + half) : i ^ 1;
        return a.layout == KVC_ROTARY_HALF ? (second ? other : i) : i >> 1;
    };
    struct Value { float y, size; };                        // (size: of its pair, 0 where nothing is turned)
    auto value = [&](int i) {
        if (i >= rotary) return Value{to_float(x[i]), 0.0f};
        int other;
        bool second;
        const int k = pair_of(i, other, second);
        const float2 cs = turn_closely(position, a.frequencies[k] * TURNS_OF_RADIANS, a.factor);
        const float f0 = to_float(x[second ? other : i]), f1 = to_float(x[second ? i : other]);
        const float y0 = f0 * cs.x - f1 * cs.y, y1 = f1 * cs.x + f0 * cs.y;
        return Value{second ? y1 : y0, position == 0.0 && a.factor == 1.0f ? 0.0f : fabsf(y0) + fabsf(y1)};
    };
    auto value_closely = [&](int i) {
        if (i >= rotary) return to_float(x[i]);
        int other;
        bool second;
        const int k = pair_of(i, other, second);
        return rotated_closely(position, a.frequencies[k], a.factor, to_float(x[second ? other : i]), to_float(x[second ? i : other]), second);
    };
    if (h < a.Hq) {                                         // (the result may lie where the query does: 32 channels and their partners are read before any is written)
        for (int i = lane; i < D; i += 32) {
            if (i >= rotary) { y[i] = x[i]; continue; }
            int other;
            bool second;
            const int k = pair_of(i, other, second);
            if (second) continue;
            const float2 cs = turn_closely(position, a.frequencies[k] * TURNS_OF_RADIANS, a.factor);
            const float f0 = to_float(x[i]), f1 = to_float(x[other]);
            y[i] = from_float<T>(f0 * cs.x - f1 * cs.y);
            y[other] = from_float<T>(f1 * cs.x + f0 * cs.y);
        }
        return;
    }
    uint32_t top = 0;
    for (int i = lane; i < D; i += 32) top = max(top, size_of(value(i).y));
    top = __reduce_max_sync(0xffffffffu, top);
    if (KIND == KVC_CODES_E4M3 && rotary > 0 && at_border(top)) {
        bool above = false;
        for (int i = lane; i < D; i += 32)
            if (size_of(value(i).y) + LAST_BITS >= border_of(top)) above |= size_of(value_closely(i)) > border_of(top);
        top = border_of(top) + (__any_sync(0xffffffffu, above) ? 1 : 0);
    }
    float inverse;
    const float s = scale_of<KIND>(top, inverse);
    for (int i = lane; i < D; i += 32) {
        const Value of = value(i);
        const float v[4] = {of.y, 0.0f, 0.0f, 0.0f};
        uint32_t c;
        if (KIND == KVC_CODES_E4M3) {
            if (codes_within(v, of.size, 0.0f, 0.0f, 0.0f, inverse, NEAR * inverse, c)) c = __nv_cvt_float_to_fp8(value_closely(i) * inverse, __NV_SATFINITE, __NV_E4M3);
        } else {
            codes_of<KIND, 1>(v, s, inverse, &c);
        }
        dst[i] = (uint8_t)c;
    }
    if (lane == 0) *scale = s;
}

// ---- rows out of pages ----------------------------------------------------------------------------------------------

struct RowsParams {
    kvc_paged_rows_args a;
    kvc_div page, units, chunks;                            // divisors: page size, units of a row, threads' shares of a token
    long long slots;
    int of_token, chunk;
};

template <int KIND> __device__ __forceinline__ void values4(uint32_t c, float s, float *v) {
    if (KIND == KVC_CODES_INT8) {
        // a byte becomes the last bits of 2^23 + 128 + code
        const uint32_t b = c ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (__uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440 + i)) - 8388736.0f) * s;
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16 * i), __NV_E4M3);
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            v[2 * i] = f.x * s; v[2 * i + 1] = f.y * s;
        }
    }
}

// A thread has 16 channels of up to CHUNK heads of a token, keys or values.  KIND 0: rows of 16 bits, copied.  HBM: 16 requests of up to 16384 tokens of 8 heads out of e4m3 (705 MB) 112 us, 6.3
// TB/s (CTAs of 256 threads 125); 777 tokens of 32 heads 8 us, latency: slots, then codes and scales.
template <typename T, int KIND>
__global__ void __launch_bounds__(CODES_THREADS) paged_rows_kernel(const __grid_constant__ RowsParams p) {
    kvc_behind();
    const kvc_paged_rows_args &a = p.a;
    const bool values = blockIdx.y;
    const int id = (int)(blockIdx.x * CODES_THREADS + threadIdx.x), group = kvc_divide(id, p.units), u = id - group * (int)(a.D / 16), n = kvc_divide(group, p.chunks);
    if (n >= a.N) return;
    const int h0 = (group - n * p.of_token) * p.chunk, heads = min(p.chunk, (int)a.Hkv - h0);
    T *out = reinterpret_cast<T *>(values ? a.v_out : a.k_out) + n * (values ? a.v_token : a.k_token) + h0 * (values ? a.v_head : a.k_head) + 16 * u;
    const long long out_head = values ? a.v_head : a.k_head;
    const int slot = a.slots[n];
    const bool there = slot >= 0 && slot < p.slots;
    if (slot >= p.slots) raise_flag(a.status, KVC_FLAG_BAD_PAGE);
    const int page = there ? kvc_divide(slot, p.page) : 0, row = there ? slot - page * (int)a.page_size : 0;
    const long long at = (values ? page * a.vp_page + row * a.vp_row + h0 * a.vp_head : page * a.kp_page + row * a.kp_row + h0 * a.kp_head) + 16 * u;
    const long long head = values ? a.vp_head : a.kp_head;
    const void *pool = values ? a.vpages : a.kpages;
    constexpr int WORDS = KIND ? 1 : 2;
    uint4 c[CHUNK][WORDS];
    float s[CHUNK];
#pragma unroll
    for (int j = 0; j < CHUNK; j++) {
        if (!there || j >= heads) continue;
        if (KIND) {
            c[j][0] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(pool) + at + j * head);
            s[j] = values ? a.scales.v[page * a.scales.v_page + (h0 + j) * a.scales.v_head + row] : a.scales.k[page * a.scales.k_page + (h0 + j) * a.scales.k_head + row];
        } else {
            const uint4 *from = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(pool) + at + j * head);
            c[j][0] = from[0];
            c[j][WORDS - 1] = from[1];
        }
    }
#pragma unroll
    for (int j = 0; j < CHUNK; j++) {
        if (j >= heads) continue;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (there && KIND) {
            float v[16];
            values4<KIND>(c[j][0].x, s[j], v);
            values4<KIND>(c[j][0].y, s[j], v + 4);
            values4<KIND>(c[j][0].z, s[j], v + 8);
            values4<KIND>(c[j][0].w, s[j], v + 12);
            lo = make_uint4(pack(v[0], v[1], T()), pack(v[2], v[3], T()), pack(v[4], v[5], T()), pack(v[6], v[7], T()));
            hi = make_uint4(pack(v[8], v[9], T()), pack(v[10], v[11], T()), pack(v[12], v[13], T()), pack(v[14], v[15], T()));
        } else if (there) {
            lo = c[j][0];
            hi = c[j][WORDS - 1];
        }
        reinterpret_cast<uint4 *>(out + j * out_head)[0] = lo;
        reinterpret_cast<uint4 *>(out + j * out_head)[1] = hi;
    }
}

bool known_codes(int codes) { return codes == KVC_CODES_INT8 || codes == KVC_CODES_E4M3; }

}  // namespace

extern "C" int kvc_rotary_store_codes(const kvc_rotary_args *args, const kvc_scales *scales, kvc_stream_t stream) {
    KVC_REQUIRE(args && scales, "kvc_rotary_store_codes: null pointer");
    CodesParams p;
    memcpy(&p.a, args, sizeof(p.a));
    memcpy(&p.s, scales, sizeof(p.s));
    kvc_rotary_args &a = p.a;
    kvc_scales &s = p.s;
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_rotary_store_codes: unknown type %d", a.type);
    KVC_REQUIRE(known_codes(s.codes), "kvc_rotary_store_codes: unknown codes %d", s.codes);
    KVC_REQUIRE(a.layout == KVC_ROTARY_HALF || a.layout == KVC_ROTARY_INTERLEAVED, "kvc_rotary_store_codes: unknown layout %d", a.layout);
    KVC_REQUIRE(a.N >= 0 && a.Hq >= 0 && a.Hkv > 0 && a.D > 0 && a.D <= 65536 && a.D % 16 == 0 && a.rotary >= 0 && a.rotary <= a.D && a.rotary % 2 == 0,
                "kvc_rotary_store_codes: bad sizes (head of %lld channels, %lld rotated)", (long long)a.D, (long long)a.rotary);
    KVC_REQUIRE(a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages >= 0 && a.n_pages * a.page_size < (1ll << 31), "kvc_rotary_store_codes: bad pool");
    if (a.N == 0) return KVC_OK;
    KVC_REQUIRE((a.Hq == 0 || (a.q && a.q_out)) && a.k && a.v && a.slots && ((a.kpages && a.vpages && s.k && s.v) || a.n_pages == 0) && (a.rotary == 0 || (a.positions && a.frequencies)),
                "kvc_rotary_store_codes: null pointer");
    KVC_REQUIRE(a.Hq < (1 << 20) && a.Hkv < (1 << 20) && a.N < (1ll << 31), "kvc_rotary_store_codes: too many heads or tokens");
    const long long H = a.Hq + 2 * a.Hkv, rows = a.N * H;
    p.page = kvc_make_div((uint32_t)a.page_size);
    p.slots = a.n_pages * a.page_size;
    // (the stride of a dimension of one, and what a part that is not there says, may be anything)
    if (a.Hq == 0) a.q = nullptr, a.q_out = nullptr;
    if (a.Hq <= 1) a.q_head = a.out_head = 0;
    if (a.N == 1 || a.Hq == 0) a.q_token = a.out_token = 0;
    if (a.Hkv == 1) a.k_head = a.v_head = a.kp_head = a.vp_head = s.k_head = s.v_head = 0;
    if (a.N == 1) a.k_token = a.v_token = 0;
    if (a.page_size == 1) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1) a.kp_page = a.vp_page = s.k_page = s.v_page = 0;
    const uintptr_t pools = reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages);
    KVC_REQUIRE(((pools | a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head) & 15) == 0, "kvc_rotary_store_codes: rows of codes must start on 16 bytes");
    KVC_REQUIRE(((reinterpret_cast<uintptr_t>(s.k) | reinterpret_cast<uintptr_t>(s.v)) & 3) == 0, "kvc_rotary_store_codes: scales must start on 4 bytes");
    // What is written in no order must not overlap: rows of the results, of a pool or of the scales each other, a result what another thread reads.  (Sizes in halves of 16 bits.)
    const kvc_rows q = kvc_make_rows(a.q, a.D, a.N, a.q_token, a.Hq, a.q_head), out = kvc_make_rows(a.q_out, a.D, a.N, a.out_token, a.Hq, a.out_head);
    const kvc_rows k = kvc_make_rows(a.k, a.D, a.N, a.k_token, a.Hkv, a.k_head), v = kvc_make_rows(a.v, a.D, a.N, a.v_token, a.Hkv, a.v_head);
    const kvc_rows written[4] = {kvc_make_rows(a.kpages, a.D / 2, a.n_pages, a.kp_page / 2, a.page_size, a.kp_row / 2, a.Hkv, a.kp_head / 2),
                                 kvc_make_rows(a.vpages, a.D / 2, a.n_pages, a.vp_page / 2, a.page_size, a.vp_row / 2, a.Hkv, a.vp_head / 2),
                                 kvc_make_rows(s.k, 2 * a.page_size, a.n_pages, 2 * s.k_page, a.Hkv, 2 * s.k_head),
                                 kvc_make_rows(s.v, 2 * a.page_size, a.n_pages, 2 * s.v_page, a.Hkv, 2 * s.v_head)};
    KVC_REQUIRE(a.Hq == 0 || out.apart, "kvc_rotary_store_codes: rows of the output overlap");
    KVC_REQUIRE(a.Hq == 0 || kvc_rows_equal(q, out) || !kvc_rows_overlap(q, out), "kvc_rotary_store_codes: the output overlaps the queries and is not them");
    KVC_REQUIRE(a.Hq == 0 || !(kvc_rows_overlap(k, out) || kvc_rows_overlap(v, out)), "kvc_rotary_store_codes: the output overlaps the keys or the values");
    for (int i = 0; i < 4; i++) {
        KVC_REQUIRE(written[i].apart, "kvc_rotary_store_codes: rows of a pool or of its scales overlap");
        for (int j = 0; j < i; j++) KVC_REQUIRE(!kvc_rows_overlap(written[i], written[j]), "kvc_rotary_store_codes: the pools or their scales overlap");
        KVC_REQUIRE(!kvc_rows_overlap(written[i], k) && !kvc_rows_overlap(written[i], v) && (a.Hq == 0 || (!kvc_rows_overlap(written[i], q) && !kvc_rows_overlap(written[i], out))),
                    "kvc_rotary_store_codes: a pool overlaps what is read or the output");
    }
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         (a.rotary ? reinterpret_cast<uintptr_t>(a.frequencies) : 0);
    const int64_t strides = a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head | a.out_token | a.out_head;
    cudaStream_t st = kvc_cu(stream);
    const bool fp16 = a.type == KVC_TYPE_FP16, whole = s.codes == KVC_CODES_INT8;
    p.units = (int)(a.D / 16);
    p.lanes = 1;
    while (p.lanes < p.units) p.lanes *= 2;
    if ((at & 15) == 0 && (strides & 7) == 0 && a.rotary % 16 == 0 && p.lanes <= 32) {
        p.parts[0] = {a.q, a.q_out, a.q_token, a.q_head, a.out_token, a.out_head, (int)a.Hq};
        p.parts[1] = {a.k, a.kpages, a.k_token, a.k_head, 0, a.kp_head, (int)a.Hkv};
        p.parts[2] = {a.v, a.vpages, a.v_token, a.v_head, 0, a.vp_head, (int)a.Hkv};
        // heads of a thread: CHUNK share its angles, unless that leaves too few threads for the device's latency
        const long long threads = (long long)CODES_CTAS * CODES_THREADS * kvc_sm_count();
        const int chunk = (int)std::max<long long>(1, std::min<long long>(CHUNK, rows * p.lanes / threads));
        p.ctas = 0;
        for (int i = 0; i < 3; i++) {
            Part &part = p.parts[i];
            const int chunks = (part.heads + chunk - 1) / chunk;
            part.chunk = chunks > 0 ? (part.heads + chunks - 1) / chunks : 1;
            part.turned = i < 2 ? (int)a.rotary / 16 : 0;
            part.first = (unsigned)p.ctas;
            p.ctas += chunks > 0 ? (part.heads + part.chunk - 1) / part.chunk : 0;
        }
        p.by_ctas = kvc_make_div((uint32_t)p.ctas);
        p.tokens = CODES_THREADS / p.lanes;
        const long long grid = (a.N + p.tokens - 1) / p.tokens * p.ctas;
        KVC_REQUIRE(grid < (1ll << 31), "kvc_rotary_store_codes: too many rows");
        auto *kernel = fp16 ? (whole ? codes_rows_kernel<__half, KVC_CODES_INT8> : codes_rows_kernel<__half, KVC_CODES_E4M3>)
                            : (whole ? codes_rows_kernel<__nv_bfloat16, KVC_CODES_INT8> : codes_rows_kernel<__nv_bfloat16, KVC_CODES_E4M3>);
        return kvc_launch_early(kernel, (unsigned)grid, CODES_THREADS, st, p);
    }
    const long long ctas = (rows + CODES_THREADS / 32 - 1) / (CODES_THREADS / 32);
    KVC_REQUIRE(ctas < (1ll << 31), "kvc_rotary_store_codes: too many rows");
    auto *kernel = fp16 ? (whole ? codes_any_kernel<__half, KVC_CODES_INT8> : codes_any_kernel<__half, KVC_CODES_E4M3>)
                        : (whole ? codes_any_kernel<__nv_bfloat16, KVC_CODES_INT8> : codes_any_kernel<__nv_bfloat16, KVC_CODES_E4M3>);
    return kvc_launch_early(kernel, (unsigned)ctas, CODES_THREADS, st, p);
}

extern "C" int kvc_paged_rows(const kvc_paged_rows_args *args, kvc_stream_t stream) {
    KVC_REQUIRE(args, "kvc_paged_rows: null pointer");
    RowsParams p;
    memcpy(&p.a, args, sizeof(p.a));
    kvc_paged_rows_args &a = p.a;
    const int codes = a.scales.codes;
    KVC_REQUIRE(a.type == KVC_TYPE_FP16 || a.type == KVC_TYPE_BF16, "kvc_paged_rows: unknown type %d", a.type);
    KVC_REQUIRE(codes == KVC_CODES_NONE || known_codes(codes), "kvc_paged_rows: unknown codes %d", codes);
    KVC_REQUIRE(a.N >= 0 && a.N < (1ll << 31) && a.Hkv > 0 && a.Hkv < (1 << 20) && a.D > 0 && a.D <= 65536 && a.D % 16 == 0, "kvc_paged_rows: bad sizes (head of %lld channels)", (long long)a.D);
    KVC_REQUIRE(a.page_size > 0 && a.page_size <= KVC_MAX_PAGE && a.n_pages >= 0 && a.n_pages * a.page_size < (1ll << 31), "kvc_paged_rows: bad pool");
    if (a.N == 0) return KVC_OK;
    KVC_REQUIRE(a.slots && a.k_out && a.v_out && ((a.kpages && a.vpages && (codes == KVC_CODES_NONE || (a.scales.k && a.scales.v))) || a.n_pages == 0), "kvc_paged_rows: null pointer");
    if (a.N == 1) a.k_token = a.v_token = 0;
    if (a.Hkv == 1) a.k_head = a.v_head = a.kp_head = a.vp_head = a.scales.k_head = a.scales.v_head = 0;
    if (a.page_size == 1) a.kp_row = a.vp_row = 0;
    if (a.n_pages <= 1) a.kp_page = a.vp_page = a.scales.k_page = a.scales.v_page = 0;
    const int64_t of_pools = a.kp_page | a.kp_row | a.kp_head | a.vp_page | a.vp_row | a.vp_head, of_rows = a.k_token | a.k_head | a.v_token | a.v_head;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.kpages) | reinterpret_cast<uintptr_t>(a.vpages) | reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out);
    KVC_REQUIRE((at & 15) == 0 && (of_rows & 7) == 0 && (of_pools & (codes == KVC_CODES_NONE ? 7 : 15)) == 0, "kvc_paged_rows: rows must start on 16 bytes");
    KVC_REQUIRE(((reinterpret_cast<uintptr_t>(a.scales.k) | reinterpret_cast<uintptr_t>(a.scales.v)) & 3) == 0, "kvc_paged_rows: scales must start on 4 bytes");
    const int64_t half = codes == KVC_CODES_NONE ? 1 : 2;   // (sizes in halves of 16 bits)
    const kvc_rows k = kvc_make_rows(a.k_out, a.D, a.N, a.k_token, a.Hkv, a.k_head), v = kvc_make_rows(a.v_out, a.D, a.N, a.v_token, a.Hkv, a.v_head);
    const kvc_rows kp = kvc_make_rows(a.kpages, a.D / half, a.n_pages, a.kp_page / half, a.page_size, a.kp_row / half, a.Hkv, a.kp_head / half);
    const kvc_rows vp = kvc_make_rows(a.vpages, a.D / half, a.n_pages, a.vp_page / half, a.page_size, a.vp_row / half, a.Hkv, a.vp_head / half);
    KVC_REQUIRE(k.apart && v.apart && !kvc_rows_overlap(k, v), "kvc_paged_rows: rows of the outputs overlap");
    const kvc_rows ks = kvc_make_rows(a.scales.k, 2 * a.page_size, a.n_pages, 2 * a.scales.k_page, a.Hkv, 2 * a.scales.k_head), vs = kvc_make_rows(a.scales.v, 2 * a.page_size, a.n_pages, 2 * a.scales.v_page, a.Hkv, 2 * a.scales.v_head);
    const kvc_rows slots = kvc_make_rows(a.slots, 2 * a.N, 1, 0, 1, 0);
    for (const kvc_rows &out : {k, v}) {
        KVC_REQUIRE(!kvc_rows_overlap(out, kp) && !kvc_rows_overlap(out, vp), "kvc_paged_rows: an output overlaps a pool");
        KVC_REQUIRE(codes == KVC_CODES_NONE || (!kvc_rows_overlap(out, ks) && !kvc_rows_overlap(out, vs)), "kvc_paged_rows: an output overlaps the scales");
        KVC_REQUIRE(!kvc_rows_overlap(out, slots), "kvc_paged_rows: an output overlaps the slots");
    }
    p.page = kvc_make_div((uint32_t)a.page_size);
    p.slots = a.n_pages * a.page_size;
    const int64_t units = a.D / 16;
    const long long threads = 4ll * CODES_THREADS * kvc_sm_count();
    const int64_t chunk = std::max<int64_t>(1, std::min<int64_t>(CHUNK, a.N * a.Hkv * units / threads)), chunks = (a.Hkv + chunk - 1) / chunk;
    p.units = kvc_make_div((uint32_t)units);
    p.chunk = (int)((a.Hkv + chunks - 1) / chunks);
    p.of_token = (int)chunks;
    p.chunks = kvc_make_div((uint32_t)chunks);
    KVC_REQUIRE(a.N * chunks * units < (1ll << 31) - CODES_THREADS, "kvc_paged_rows: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.N * chunks * units + CODES_THREADS - 1) / CODES_THREADS), 2);
    cfg.blockDim = dim3(CODES_THREADS);
    cfg.stream = kvc_cu(stream);
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    const bool fp16 = a.type == KVC_TYPE_FP16;
    auto *kernel = codes == KVC_CODES_NONE ? paged_rows_kernel<__half, 0>                          // (copied, whatever they are)
                   : codes == KVC_CODES_INT8 ? (fp16 ? paged_rows_kernel<__half, KVC_CODES_INT8> : paged_rows_kernel<__nv_bfloat16, KVC_CODES_INT8>)
                                             : (fp16 ? paged_rows_kernel<__half, KVC_CODES_E4M3> : paged_rows_kernel<__nv_bfloat16, KVC_CODES_E4M3>);
    KVC_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, (const RowsParams)p));
    return KVC_OK;
}
