// The 8-bit cache's pages: their order in memory, their scale and codes.
//
// A block is one KV head's share of a page: 16 rows of 256 values, K and V
// apart.  A full block is held as codes c in [-127, 127] (a byte c + 128 each)
// and one scale s; a value is c s.  A sequence's open block (its last page,
// not full) is held in FP16, in the same order.
//
// Scale: s = m 2^e, m in 8..15 and e >= -24, the smallest with 127 s >= the
// block's largest magnitude, and at most 512; c = x / s rounded to the
// nearest, ties to even, within [-127, 127].  Why four significant bits: c has
// seven, so c s has eleven and no bit below 2^-24, which makes it an FP16 number
// (127 * 512 = 65024 is the largest).  A block's values go into the matrix
// cores as they are, with no rounding besides the code's own, and no scale has
// to be carried along for V.  The price is a scale up to 1/8 larger than the
// smallest one, so a step at most 1/8 wider.  And the codes do not depend on
// the arithmetic: x / s = X 2^c / m with integers X < 2^11 and m < 2^4, so it is
// either exactly half-way between two codes (and then an FP32 number) or
// further from half-way, 2^c / 2m at least, than an FP32 rounding, 2^(c-13) /
// m at most, can move it.  The same holds for amax / 127 against the border
// between two scales (amax = 127 s exactly, or off by 2^-11 of it).
//
// A value that is not finite has no code.  A row of a head in which K or V
// holds one is kept as a key of NaN and a value of zeros, so that whoever sees
// the row gets NaN and whoever does not (p = 0) gets nothing of it; a full
// block with such a row has the scale NaN for K (every row of the block reads
// as NaN) and codes of the finite rows for V.
//
// Order ("page order"), made for the matrix cores' operands, so that a wave
// reads a block in four 1 KB loads of 16 bytes a lane and holds its operands:
//   K: [16 chunks of 16 dims][16 rows][16 dims]: lane l's 16 bytes of load i
//      are row l % 16, dims 64 i + 16 (l / 16) .. + 15: two k-steps of A of a
//      16x16x32 product (any k order does, as long as B has the same);
//   V: [4 groups of 4 dim tiles][64 lanes][4 tiles][4 rows]: lane l's 16 bytes
//      of load j are dims 16 (4 j + 0..3) + l % 16, rows 4 (l / 16) .. + 3: A = V^T
//      of four 16x16x16 products.
#pragma once

#include "k_common.h"
#include "kva_internal.h"

namespace kva {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int k_at(int row, int dim) { return (dim >> 4) * 256 + row * 16 + (dim & 15); }
__device__ __forceinline__ int v_at(int row, int dim) {
    const int tile = dim >> 4;
    return (tile >> 2) * 1024 + ((row >> 2) * 16 + (dim & 15)) * 16 + (tile & 3) * 4 + (row & 3);
}

// Two codes as FP16 integers: the bytes u = c + 128 under 0x64 are 1024 + u,
// and 1152 less is c, exactly.
__device__ __forceinline__ uint32_t add_h2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, a) + __builtin_bit_cast(half2_t, b));
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, a) * __builtin_bit_cast(half2_t, b));
}
constexpr uint32_t kMinus1152 = 0xe480e480u;  // FP16 pair (-1152, -1152)
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
    return add_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), kMinus1152);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
    return add_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u), kMinus1152);
}
// Eight codes as the integers they are (an operand of 16x16x32 products).
__device__ __forceinline__ uint4 codes8(uint32_t w0, uint32_t w1) {
    return make_uint4(codes_lo(w0), codes_hi(w0), codes_lo(w1), codes_hi(w1));
}
// Four codes times the scale pair s2: exact, see above.
__device__ __forceinline__ uint2 values4(uint32_t w, uint32_t s2) {
    return make_uint2(mul_h2(codes_lo(w), s2), mul_h2(codes_hi(w), s2));
}
__device__ __forceinline__ uint32_t scale_h2(float s) {
    const uint32_t h = f2h(s);  // exact: four significant bits, 2^-21 .. 512 (or 0)
    return h | (h << 16);
}

__device__ __forceinline__ bool not_finite(uint32_t pair) {
    return (pair & 0x7c00u) == 0x7c00u || (pair & 0x7c000000u) == 0x7c000000u;
}

// The scale of a block whose largest magnitude is amax.
__device__ __forceinline__ float block_scale(float amax) {
    const float t = amax / 127.0f;
    const float s = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, t) + 0xfffffu) & 0xfff00000u);
    return fminf(fmaxf(s, 0x1p-21f), 512.0f);
}
// The byte of value x in a block of scale s.
__device__ __forceinline__ uint32_t code_of(float x, float s) {
    const float c = fminf(fmaxf(rintf(x / s), -127.0f), 127.0f);
    return static_cast<uint32_t>(static_cast<int>(c) + 128);
}

// Rows of a block by half-waves (512 threads, half-wave r has row r), each
// lane dims 8 (lane % 32) .. + 7 as FP16.
struct BlockRow {
    uint4 k, v;
};

__device__ __forceinline__ void mend_row(BlockRow &x) {
    const bool bad = not_finite(x.k.x) || not_finite(x.k.y) || not_finite(x.k.z) || not_finite(x.k.w) ||
                     not_finite(x.v.x) || not_finite(x.v.y) || not_finite(x.v.z) || not_finite(x.v.w);
    const uint64_t all = __ballot(bad);
    if ((threadIdx.x & 32) ? (all >> 32) != 0 : (all & 0xffffffffull) != 0) {
        x.k = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u);
        x.v = make_uint4(0, 0, 0, 0);
    }
}

// Row `row` of an open block to or from memory in page order.
__device__ __forceinline__ void store_open_row(uint16_t *block, int row, int l32, const BlockRow &x) {
    st16(block + k_at(row, 8 * l32), x.k);
    const uint32_t w[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
    uint16_t *v = block + kPageElems;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[v_at(row, 8 * l32 + i)] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
}
__device__ __forceinline__ BlockRow load_open_row(const uint16_t *block, int row, int l32) {
    BlockRow x;
    x.k = ld16(block + k_at(row, 8 * l32));
    const uint16_t *v = block + kPageElems;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 1] |= static_cast<uint32_t>(v[v_at(row, 8 * l32 + i)]) << (16 * (i & 1));
    x.v = make_uint4(w[0], w[1], w[2], w[3]);
    return x;
}
// Row `row` of a full block, as the FP16 numbers that its codes stand for.
__device__ __forceinline__ BlockRow load_code_row(const uint8_t *k, const uint8_t *v, const float *scales, int row,
                                                  int l32) {
    const float2 s = *reinterpret_cast<const float2 *>(scales);
    const uint32_t ks = scale_h2(s.x), vs = scale_h2(s.y);  // NaN stays NaN
    const uint2 kc = *reinterpret_cast<const uint2 *>(k + k_at(row, 8 * l32));
    uint32_t vc[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) vc[i >> 2] |= static_cast<uint32_t>(v[v_at(row, 8 * l32 + i)]) << (8 * (i & 3));
    const uint2 k0 = values4(kc.x, ks), k1 = values4(kc.y, ks), v0 = values4(vc[0], vs), v1 = values4(vc[1], vs);
    BlockRow x;
    x.k = make_uint4(k0.x, k0.y, k1.x, k1.y);
    x.v = make_uint4(v0.x, v0.y, v1.x, v1.y);
    return x;
}

struct CloseLds {
    float2 amax[16];
    uint32_t bad;
    uint8_t v[kPageElems];
};

// Sixteen rows, one per half-wave of a 512-thread workgroup, as codes in the
// block at k, v, scales.  Ends with every wave past its LDS reads but not
// synchronised; every thread of the workgroup calls it.
__device__ __forceinline__ void close_block(const BlockRow &x, uint8_t *k, uint8_t *v, float *scales, CloseLds &lds) {
    const int row = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const uint32_t kw[4] = {x.k.x, x.k.y, x.k.z, x.k.w}, vw[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
    const bool bad = not_finite(kw[0]);  // a row is NaN as a whole (mend_row)
    float ka = 0.0f, va = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ka = fmaxf(ka, fmaxf(fabsf(lo_f(kw[i])), fabsf(hi_f(kw[i]))));
        va = fmaxf(va, fmaxf(fabsf(lo_f(vw[i])), fabsf(hi_f(vw[i]))));
    }
    if (threadIdx.x == 0) lds.bad = 0;
    __syncthreads();
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        ka = fmaxf(ka, __shfl_xor(ka, o));
        va = fmaxf(va, __shfl_xor(va, o));
    }
    if (l32 == 0) {
        lds.amax[row] = make_float2(ka, va);
        if (bad) atomicOr(&lds.bad, 1u);
    }
    __syncthreads();
    ka = va = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        ka = fmaxf(ka, lds.amax[r].x);
        va = fmaxf(va, lds.amax[r].y);
    }
    const float ks = block_scale(ka), vs = block_scale(va);
    const bool spoilt = lds.bad != 0;
    uint32_t kc[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t h = kw[i >> 1], g = vw[i >> 1];
        const float xk = (i & 1) ? hi_f(h) : lo_f(h), xv = (i & 1) ? hi_f(g) : lo_f(g);
        kc[i >> 2] |= (spoilt ? 128u : code_of(xk, ks)) << (8 * (i & 3));
        lds.v[v_at(row, 8 * l32 + i)] = static_cast<uint8_t>(code_of(xv, vs));
    }
    *reinterpret_cast<uint2 *>(k + k_at(row, 8 * l32)) = make_uint2(kc[0], kc[1]);
    if (threadIdx.x == 0)
        *reinterpret_cast<float2 *>(scales) =
            make_float2(spoilt ? __builtin_nanf("") : ks, vs);
    __syncthreads();
    reinterpret_cast<uint2 *>(v)[threadIdx.x] = reinterpret_cast<const uint2 *>(lds.v)[threadIdx.x];
}

}  // namespace kva
