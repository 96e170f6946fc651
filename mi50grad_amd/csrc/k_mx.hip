// Rows as microscaled rows and back, the order in which the products take
// 4-bit weights, and the norm that leaves microscaled rows (gfx950).
//
// All of it is bound by memory where there is enough: bytes are read and written
// once, a lane taking 16 bytes of fp16 (a large copy runs at 4.8 TB/s here; what
// the last kernel left in the caches is read faster).  A few rows take what a
// launch takes, 1.4 to 2.5 us.
#include "k_mx.h"
#include "kva_internal.h"

namespace kva {
namespace {

constexpr int kMxThreads = 256;

__device__ __forceinline__ void half8_to_float(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = lo_f(w[i]);
        x[2 * i + 1] = hi_f(w[i]);
    }
}

// A lane takes eight values of a row, four lanes a block.  5120 x 6144 to 4 bits:
// 18.5 us, 4.3 TB/s (two pieces of a lane on their way: the same).
template <int BITS>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(MxRows a) {
    const uint32_t per_row = a.cols / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kMxThreads + threadIdx.x;
    if (i >= a.rows * static_cast<int64_t>(per_row)) return;  // whole quads leave
    const int64_t row = i / per_row;
    const uint32_t c8 = static_cast<uint32_t>(i - row * per_row);
    float x[8];
    half8_to_float(ld16(a.x + row * a.x_stride + 8 * c8), x);
    mx_store_quad<BITS>(x, a.codes, a.scales, static_cast<size_t>(i) * 8);
}

// A lane gives eight values.  5120 x 6144 of 4 bits: 12.8 us, 6.2 TB/s, with the
// codes in the caches; 8192 x 5120 of 8 bits: 20 us, 6.3 TB/s.
template <int BITS>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(MxRows a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kMxThreads + threadIdx.x;
    if (i >= a.rows * static_cast<int64_t>(a.cols / 8)) return;
    const uint32_t byte = a.scales[i / 4];
    const float s = mx_scale(byte);
    half2_t v[4];
    if constexpr (BITS == 8) {
        const uint2 c = *reinterpret_cast<const uint2 *>(a.codes + 8 * i);
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(c.x), s, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(c.x), s, true);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(c.y), s, false);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(c.y), s, true);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(a.codes + 4 * i);
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = byte == kMxNan ? 0x7e007e00u : __builtin_bit_cast(uint32_t, v[j]);
    st16(a.y + 8 * i, make_uint4(o[0], o[1], o[2], o[3]));
}

// Weight rows in the order of the products' A operand (MxWeight): lane l of a
// wave takes row l % 32's 16 bytes of block 2 * step + l / 32.  Rows past the
// last are zeros.  A wave moves four steps (256 values of 32 rows), and with
// them the dword of scales that each lane needs for those.  Weights are packed
// once: 12288 x 5120 in 23 us, 2.9 TB/s, where a copy of as much takes 14.
__global__ __launch_bounds__(kMxThreads) void mx_pack_kernel(MxPack a) {
    const int lane = threadIdx.x & 63;
    const int n_quad = a.cols / 256;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (kMxThreads / 64) + (threadIdx.x >> 6);
    const int64_t tile = w / n_quad;
    const int quad = static_cast<int>(w - tile * n_quad);
    if (tile >= a.n_tiles) return;
    const int64_t row = tile * 32 + (lane & 31);
    const int half = lane >> 5;
    const bool in = row < a.rows;
    uint4 c[4];
    uint32_t scales = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int block = 8 * quad + 2 * s + half;
        c[s] = in ? *reinterpret_cast<const uint4 *>(a.codes + row * (a.cols / 2) + 16 * block) : make_uint4(0, 0, 0, 0);
        const uint32_t b = in ? a.scales[row * (a.cols / 32) + block] : 1u;
        scales |= b << (8 * s);
    }
    uint8_t *dst = a.packed + (tile * (a.cols / 64) + 4 * quad) * 1024 + 16 * lane;
#pragma unroll
    for (int s = 0; s < 4; ++s) *reinterpret_cast<uint4 *>(dst + 1024 * s) = c[s];
    uint8_t *sc = a.packed + a.n_tiles * 32 * static_cast<int64_t>(a.cols / 2);
    *reinterpret_cast<uint32_t *>(sc + (tile * n_quad + quad) * 256 + 4 * lane) = scales;
}

// hidden + delta (rounded to fp16: the residual stream's type) and its norm,
// x = s / sqrt(mean(s^2) + eps) * w over the rounded sums, rounded once to what
// is asked for.  A workgroup takes a row and holds it in registers, so every
// byte is read once; lanes past the row hold zeros.  8192 x 5120 to 8 bits: 59
// us, 5.0 TB/s; 2048 x 5120 to fp16: 14.5 us, 5.8 TB/s.
template <int BITS, int PER>
__global__ __launch_bounds__(1024) void add_rmsnorm_kernel(MxNorm a) {
    __shared__ float red[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const size_t row = static_cast<size_t>(blockIdx.x) * a.cols;
    uint4 h[PER], d[PER], w[PER];
    const bool add = a.delta != nullptr;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t c = 8 * (threadIdx.x + j * blockDim.x);
        const bool in = c < static_cast<uint32_t>(a.cols);
        h[j] = in ? ld16(a.hidden + row + c) : make_uint4(0, 0, 0, 0);
        d[j] = in && add ? ld16(a.delta + row + c) : make_uint4(0, 0, 0, 0);
        w[j] = in ? ld16(a.w + c) : make_uint4(0, 0, 0, 0);
    }
    float x[PER][8], sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        half8_to_float(h[j], x[j]);
        if (add) {
            // In fp16: one rounding (through fp32 a small term can be lost
            // before a tie is decided).
            h[j] = __builtin_bit_cast(uint4, __builtin_bit_cast(half8_t, h[j]) + __builtin_bit_cast(half8_t, d[j]));
            half8_to_float(h[j], x[j]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[j][i], x[j][i], sum);
    }
    if (add) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t c = 8 * (threadIdx.x + j * blockDim.x);
            if (c < static_cast<uint32_t>(a.cols)) st16(a.sum_out + row + c, h[j]);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    float all = 0.f;
    for (int i = 0; i < waves; ++i) all += red[i];
    const float inv = 1.0f / sqrtf(all / static_cast<float>(a.cols) + a.eps);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t c = 8 * (threadIdx.x + j * blockDim.x);
        float g[8];
        half8_to_float(w[j], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = x[j][i] * inv * g[i];
        if (c >= static_cast<uint32_t>(a.cols)) continue;  // whole quads
        if constexpr (BITS == 16) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = pack_h2(x[j][2 * i], x[j][2 * i + 1]);
            st16(static_cast<uint16_t *>(a.out) + row + c, make_uint4(o[0], o[1], o[2], o[3]));
        } else {
            mx_store_quad<BITS>(x[j], static_cast<uint8_t *>(a.out), a.scales, row + c);
        }
    }
}

template <int BITS>
hipError_t norm_of(const MxNorm &a, hipStream_t s) {
    const int lanes = (a.cols / 8 + 63) / 64 * 64;
    const int per = (lanes + 1023) / 1024;
    const dim3 grid(static_cast<unsigned>(a.n_tok)), block((lanes / per + 63) / 64 * 64);
    if (per == 1) hipLaunchKernelGGL((add_rmsnorm_kernel<BITS, 1>), grid, block, 0, s, a);
    else if (per == 2) hipLaunchKernelGGL((add_rmsnorm_kernel<BITS, 2>), grid, block, 0, s, a);
    else if (per <= 4) hipLaunchKernelGGL((add_rmsnorm_kernel<BITS, 4>), grid, dim3(1024), 0, s, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantize(const MxRows &a, int bits, hipStream_t s) {
    const int64_t lanes = a.rows * static_cast<int64_t>(a.cols / 8);
    const dim3 grid(static_cast<unsigned>((lanes + kMxThreads - 1) / kMxThreads)), block(kMxThreads);
    if (bits == 8) hipLaunchKernelGGL(mx_quantize_kernel<8>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(mx_quantize_kernel<4>, grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const MxRows &a, int bits, hipStream_t s) {
    const int64_t lanes = a.rows * static_cast<int64_t>(a.cols / 8);
    const dim3 grid(static_cast<unsigned>((lanes + kMxThreads - 1) / kMxThreads)), block(kMxThreads);
    if (bits == 8) hipLaunchKernelGGL(mx_dequantize_kernel<8>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(mx_dequantize_kernel<4>, grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_mx_pack(const MxPack &a, hipStream_t s) {
    const int64_t waves = a.n_tiles * (a.cols / 256);
    const int per = kMxThreads / 64;
    hipLaunchKernelGGL(mx_pack_kernel, dim3(static_cast<unsigned>((waves + per - 1) / per)), dim3(kMxThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_add_rmsnorm(const MxNorm &a, int bits, hipStream_t s) {
    return bits == 16 ? norm_of<16>(a, s) : bits == 8 ? norm_of<8>(a, s) : norm_of<4>(a, s);
}

}  // namespace kva
