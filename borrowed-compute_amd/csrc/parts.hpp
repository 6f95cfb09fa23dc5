// Operands of the f16 matrix cores in two parts, for attention whose results are to be as near as
// f32 arithmetic comes: q and the softmax weights are f16 values and the rests of their rounding, 22
// bits together, every product exact, sums in f32. Shared by the kernels over 4-bit caches and those
// over pages.
//
// The running maximum is a reference 2^11 under it, raised only where a weight would pass 2^15:
// weights stay within an f16, their low parts well above its smallest, and most tiles raise nothing.
#pragma once

#include "common.hpp"

namespace bchip {

constexpr float W_BIAS = 11.0f;  // log2 of the weight of a row's largest score when ref is set
constexpr float W_MOST = 15.0f;  // of any weight: an f16 holds it

// The larger of two, a number before a NaN: fmaxf without the quieting of its operands.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The largest magnitude of them and `top`.
__device__ __forceinline__ float q_top(const float (&x)[8], float top) {
#pragma unroll
    for (int i = 0; i < 8; i++) top = larger(top, fabsf(x[i]));
    return top;
}

// From a row's largest |q|: q times k is q scale log2 e brought to 2^13 .. 2^14, c takes it back.
__device__ __forceinline__ void q_scale(float top, float sc, float& k, float& c) {
    int e = (int)(__float_as_uint(top * fabsf(sc)) >> 23) - 127;  // (of an infinity 128: its row is NaN)
    e = e < -100 ? -100 : e;
    k = sc * __uint_as_float((uint32_t)(13 - e + 127) << 23);
    c = __uint_as_float((uint32_t)(e - 13 + 127) << 23);
}

__device__ __forceinline__ void q_parts(const float (&x)[8], float k, half8& hi, half8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const half2 h = __builtin_convertvector((f32x2{x[i] * k, x[i + 1] * k}), half2);
        const half2 r = __builtin_convertvector((f32x2{__builtin_fmaf(x[i], k, -(float)h[0]), __builtin_fmaf(x[i + 1], k, -(float)h[1])}), half2);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = r[0], lo[i + 1] = r[1];
    }
}

// A row's scores are c s (c a power of two), its weights 2^(c s - ref). Where some score of these
// 16 N slots passes ref by more than W_MOST, the refs rise to W_BIAS under their rows' maxima (to
// the maxima themselves where those are so large that the difference would be lost), and what
// was summed against the old one is to be multiplied by f.
template <int N>
__device__ __forceinline__ bool raise(const f32x4 (&s)[N], float c, float& ref, float& f) {
    float top = larger(larger(s[0][0], s[0][1]), larger(s[0][2], s[0][3]));
    if constexpr (N == 2) top = larger(top, larger(larger(s[1][0], s[1][1]), larger(s[1][2], s[1][3])));
    top *= c;
    if (!__any(top > ref + W_MOST)) return false;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float to = fmaxf(ref, fabsf(top) < 0x1p23f ? top - W_BIAS : top);
    f = to == -INFINITY ? 1.0f : exp2_hw(ref - to);
    ref = to;
    return true;
}

// The weights' B operand, the rounded values (hi) and the rest (lo); their sum goes to l. With
// PART, hi comes back as the rounded values times 1 - keep plus the rest times keep (0 or 1): a
// lane holds one part.
template <bool PART>
__device__ __forceinline__ void weights(const f32x4 (&s)[2], float c, float ref, float keep, float& l, half8& hi, half8& lo) {
    const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float w0 = exp2_hw(__builtin_fmaf(s[i >> 2][i & 3], c, -base));
        const float w1 = exp2_hw(__builtin_fmaf(s[i >> 2][(i & 3) + 1], c, -base));
        l += w0;
        l += w1;
        const half2 h = __builtin_convertvector((f32x2{w0, w1}), half2);
        const float k = PART ? -keep : -1.0f;
        const half2 r = __builtin_convertvector((f32x2{__builtin_fmaf((float)h[0], k, w0), __builtin_fmaf((float)h[1], k, w1)}), half2);
        hi[i] = PART ? r[0] : h[0];
        hi[i + 1] = PART ? r[1] : h[1];
        lo[i] = r[0];
        lo[i + 1] = r[1];
    }
}

__device__ __forceinline__ float ror8(float x) {  // lane n of each 16 gets lane (n + 8) % 16's
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
}

}  // namespace bchip
