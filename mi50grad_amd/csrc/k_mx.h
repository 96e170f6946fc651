// Microscaled rows (gfx950): blocks of 32 elements with one scale.
//
// An element is 8 bits (sign, 4 exponent bits of bias 7, 3 mantissa bits; the
// largest value is 448) or 4 bits (sign, 2 exponent bits of bias 1, 1 mantissa
// bit; the largest is 6), a scale is the byte b of 2^(b - 127): what the
// scaled matrix instructions take.  A block's scale is the smallest power of
// two, from 2^-126 on, for which the largest element covers its largest
// magnitude, so nothing saturates (taking the exponent of the largest
// magnitude instead would cut a 4-bit block's largest value by up to a
// quarter, 8 clipped to 6).  Elements are x / scale rounded to the nearest,
// ties to even, in one step from what x is held in.  A block with a value
// that is not finite has the scale byte 255, which products and reads take as
// NaN, and zero elements.
#pragma once

#include "k_common.h"

namespace kva {

constexpr uint32_t kMxNan = 255;

typedef short short2_t __attribute__((ext_vector_type(2)));

// The scale byte for a block of largest magnitude amax (finite): with the
// largest element m 2^e, amax's exponent less e, and one more where its
// significand is above m.  Bits below 1 (2^-126) are taken as 1, so that the
// scale is a normal fp32 number.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(float amax) {
    constexpr uint32_t kMant = BITS == 8 ? 0x600000u : 0x400000u;  // 1.75, 1.5
    constexpr int kExp = BITS == 8 ? 8 : 2;
    const int b = static_cast<int>((__builtin_bit_cast(uint32_t, amax) + (0x7fffffu - kMant)) >> 23) - kExp;
    return static_cast<uint32_t>(max(b, 1));
}

// The scale of byte b below 255; of 0, 2^-127, a subnormal.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __builtin_bit_cast(float, byte == 0 ? 0x400000u : byte << 23);
}

// Eight values as elements of scale s, the first in the lowest bits.
__device__ __forceinline__ uint2 mx_encode8(const float (&x)[8], float s) {
    short2_t r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        r[i] = short2_t{0, 0};
        r[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r[i], x[4 * i], x[4 * i + 1], s, false);
        r[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r[i], x[4 * i + 2], x[4 * i + 3], s, true);
    }
    return make_uint2(__builtin_bit_cast(uint32_t, r[0]), __builtin_bit_cast(uint32_t, r[1]));
}
__device__ __forceinline__ uint32_t mx_encode4(const float (&x)[8], float s) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], s, 3);
    return r;
}

// The largest magnitude of a block that four neighbouring lanes hold, as the
// bits of an fp32 magnitude (NaN above infinity above all finite ones).
__device__ __forceinline__ uint32_t quad_max_u(uint32_t x) {
    x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kDppQuadXor1, 0xF, 0xF, false)));
    return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kDppQuadXor2, 0xF, 0xF, false)));
}

// A quad's block: each lane's eight values as elements at codes + at * BITS /
// 8 (`at`: index of the lane's first value in the row-major array, a multiple
// of 8) and the scale byte at scales[at / 32], written by the quad's first lane.
template <int BITS>
__device__ __forceinline__ void mx_store_quad(const float (&x)[8], uint8_t *codes, uint8_t *scales, size_t at) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
    m = quad_max_u(m);
    const bool fine = m < 0x7f800000u;
    const uint32_t byte = fine ? mx_scale_byte<BITS>(__builtin_bit_cast(float, m)) : kMxNan;
    const float s = mx_scale(byte);
    if constexpr (BITS == 8) {
        const uint2 c = mx_encode8(x, s);
        *reinterpret_cast<uint2 *>(codes + at) = fine ? c : make_uint2(0, 0);
    } else {
        const uint32_t c = mx_encode4(x, s);
        *reinterpret_cast<uint32_t *>(codes + at / 2) = fine ? c : 0u;
    }
    if (at % 32 == 0) scales[at / 32] = static_cast<uint8_t>(byte);
}

}  // namespace kva
