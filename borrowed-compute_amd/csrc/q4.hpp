// The 4-bit cache format (BCHIP_Q4), shared by the kernels that write, move and read it.
//
// A buffer is an array of units of 256 consecutive elements, 144 bytes each: 128 bytes of codes
// (two a byte, the even element in the low four bits), then the f16 scales of the unit's eight
// blocks of 32. An element is (code - 8) * scale. A block's scale d is the value of its largest
// magnitude over -8 (the positive one of two equal ones, so code 0 is that value), rounded to 7
// significant bits and held within 2^-14 .. 896; a block with an element that is not finite has
// the scale NaN.
//
// Seven bits, because a value is then exactly an f16, (code - 8) d taking at most 3 + 7
// significant bits, and one packed f16 FMA makes two of them: with the code in bits 4 .. 7 of a
// half whose exponent says 64, that half is 64 + code, and (64 + code) d - 72 d rounds nothing,
// 72 d taking 4 + 7 bits. The bounds keep 72 d within f16's range and every value but 0 a normal
// f16. A scale's rounding moves a value by at most 2^-7 of itself, beside the codes' steps of
// an eighth of the block's largest.
#pragma once

#include "common.hpp"

namespace bchip {

constexpr uint32_t Q4_UNIT = 256;        // elements a unit
constexpr uint32_t Q4_UNIT_BYTES = 144;  // its bytes
constexpr uint32_t Q4_BLOCK = 32;        // elements that share a scale

// Byte offset of element e's code (e even: of the byte that holds e and e + 1).
__host__ __device__ __forceinline__ uint64_t q4_code_at(uint64_t e) {
    return (e >> 8) * Q4_UNIT_BYTES + ((e & 255) >> 1);
}
// Byte offset of the scale of element e's block.
__host__ __device__ __forceinline__ uint64_t q4_scale_at(uint64_t e) {
    return (e >> 8) * Q4_UNIT_BYTES + 128 + ((e & 255) >> 5) * 2;
}
// The same within 32 bits, for elements of one tile.
__device__ __forceinline__ uint32_t q4_code_at32(uint32_t e) { return (e >> 8) * Q4_UNIT_BYTES + ((e & 255) >> 1); }
__device__ __forceinline__ uint32_t q4_scale_at32(uint32_t e) {
    return (e >> 8) * Q4_UNIT_BYTES + 128 + ((e & 255) >> 5) * 2;
}

// Sixteen consecutive lanes quantise a block, each two consecutive elements of it: the block's
// scale, and the byte of this lane's codes. Every lane of the sixteen must be active.
__device__ __forceinline__ f16 q4_quantise(float x0, float x1, uint8_t& codes) {
    // Magnitude bits over the sign (1 for positive): the largest key is the largest magnitude,
    // the positive one of two.
    const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
    uint32_t key = max((b0 << 1) | (~b0 >> 31), (b1 << 1) | (~b1 >> 31));
#pragma unroll
    for (int d = 1; d < 16; d *= 2) key = max(key, (uint32_t)__shfl_xor((int)key, d, 16));
    if ((key >> 1) >= 0x7f800000u) {  // an infinity or a NaN
        codes = 0x88;
        return __builtin_bit_cast(f16, (uint16_t)0x7e00);
    }
    uint32_t u = __float_as_uint(__uint_as_float(key >> 1) * 0.125f);
    u = (u + 0xffffu + ((u >> 17) & 1u)) & ~0x1ffffu;  // 7 significant bits, to nearest even
    float d = fminf(fmaxf(__uint_as_float(u), 0x1p-14f), 896.0f);
    if (key & 1u) d = -d;
    const float r = 1.0f / d;
    const float n0 = fminf(fmaxf(rintf(x0 * r), -8.0f), 7.0f), n1 = fminf(fmaxf(rintf(x1 * r), -8.0f), 7.0f);
    codes = (uint8_t)((uint32_t)((int)n0 + 8) | (uint32_t)((int)n1 + 8) << 4);
    return (f16)d;
}

}  // namespace bchip
