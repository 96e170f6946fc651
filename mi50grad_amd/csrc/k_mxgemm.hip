// The projections by 4-bit weights (gfx950): microscaled rows of activations
// in 8 or 4 bits against packed 4-bit weight rows,
//   Y[t][n] = sum_k X[t][k] W[n][k],
// on v_mfma_scale_f32_32x32x64_f8f6f4 with weight rows as A and tokens as B:
// the products of a block of 32 are taken exactly, times both scales, and
// summed in fp32.  Lane l holds of A row l % 32's block l / 32 of a step of 64
// (16 bytes), of an 8-bit B token l % 32's bytes 16 (l / 32) .. +15 of either
// block (the instruction's order for 8 bits), of a 4-bit B its block l / 32,
// and of both one scale byte, of block l / 32.
#include "k_mx.h"
#include "kva_internal.h"

namespace kva {
namespace {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kMxWaves = 4;

template <int BITS, int SEL>
__device__ __forceinline__ float16_t mx_mfma(int8v_t w, int8v_t x, float16_t c, uint32_t ws, uint32_t xs) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 4, BITS == 8 ? 0 : 4, SEL, ws, 0, xs);
}

// A wave takes 32 weight rows and 32 tokens, straight from memory, and leaves
// fp32 partials [token][row] for a finish kernel.
template <int BITS>
__global__ __launch_bounds__(64 * kMxWaves) void mx_part_kernel(ProjectArgs a, MxProduct m) {
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int N = a.n_a + a.n_b;
    const int n_rt = (N + 31) / 32, n_mt = (a.n_tok + 31) / 32;
    const int tile = blockIdx.x * kMxWaves + (threadIdx.x >> 6);
    if (tile >= n_rt * n_mt) return;
    const int rt = tile / n_mt, mt = tile - rt * n_mt;
    const int K = a.hidden, steps = K / 64;
    const int rta = a.n_a / 32;
    const bool first = rt < rta || a.n_b == 0;
    const uint8_t *wp = first ? m.w_a : m.w_b;
    const int64_t wt = first ? rt : rt - rta, w_tiles = ((first ? a.n_a : a.n_b) + 31) / 32;
    const uint8_t *wc = wp + wt * steps * 1024 + 16 * lane;
    const uint8_t *wsc = wp + w_tiles * 16 * K + wt * (steps / 4) * 256 + 4 * lane;
    const int t = min(32 * mt + col, a.n_tok - 1);
    const uint8_t *xc = m.x + static_cast<size_t>(t) * (K * BITS / 8) + 16 * half;
    const uint8_t *xsc = m.x_scales + static_cast<size_t>(t) * (K / 32) + half;
    float16_t acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto step = [&](auto sel, int s, uint32_t ws) {
        const uint4 w = *reinterpret_cast<const uint4 *>(wc + 1024 * s);
        const uint4 x0 = *reinterpret_cast<const uint4 *>(xc + (BITS == 8 ? 64 : 32) * s);
        uint4 x1 = make_uint4(0, 0, 0, 0);
        if constexpr (BITS == 8) x1 = *reinterpret_cast<const uint4 *>(xc + 64 * s + 32);
        const uint32_t xs = xsc[2 * s];
        const int8v_t wv = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
        const int8v_t xv = {static_cast<int>(x0.x), static_cast<int>(x0.y), static_cast<int>(x0.z), static_cast<int>(x0.w),
                            static_cast<int>(x1.x), static_cast<int>(x1.y), static_cast<int>(x1.z), static_cast<int>(x1.w)};
        acc = mx_mfma<BITS, decltype(sel)::value>(wv, xv, acc, ws, xs);
    };
    for (int q = 0; q < steps / 4; ++q) {
        const uint32_t ws = *reinterpret_cast<const uint32_t *>(wsc + 256 * q);
        step(std::integral_constant<int, 0>{}, 4 * q, ws);
        step(std::integral_constant<int, 1>{}, 4 * q + 1, ws);
        step(std::integral_constant<int, 2>{}, 4 * q + 2, ws);
        step(std::integral_constant<int, 3>{}, 4 * q + 3, ws);
    }
    if (32 * mt + col >= a.n_tok) return;
    float *part = a.part + static_cast<size_t>(32 * mt + col) * N + 32 * rt + 4 * half;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (32 * rt + 8 * i + 4 * half < N)
            *reinterpret_cast<float4_t *>(part + 8 * i) = float4_t{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
}

}  // namespace

bool plan_mx(const ProjectArgs &a, const MxProduct &m, bool heads, int n_cu, size_t part_floats, ProductPlan &plan) {
    plan = ProductPlan{};
    plan.partial = true;
    plan.splits = 1;
    plan.bm = plan.bn = 32;
    plan.form = plan.pair = -1;
    return static_cast<size_t>(a.n_tok) * (a.n_a + a.n_b) <= part_floats;
}

hipError_t launch_mx_product(const ProjectArgs &args, const MxProduct &m, bool heads, const ProductPlan &plan,
                             hipStream_t s) {
    ProjectArgs a = args;
    a.splits = plan.splits;
    hipError_t e = a.ev_before ? hipEventRecord(a.ev_before, s) : hipSuccess;
    if (e != hipSuccess) return e;
    const int64_t tiles = static_cast<int64_t>((a.n_a + a.n_b + 31) / 32) * ((a.n_tok + 31) / 32);
    const dim3 grid(static_cast<unsigned>((tiles + kMxWaves - 1) / kMxWaves)), block(64 * kMxWaves);
    if (m.bits == 8) hipLaunchKernelGGL(mx_part_kernel<8>, grid, block, 0, s, a, m);
    else hipLaunchKernelGGL(mx_part_kernel<4>, grid, block, 0, s, a, m);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (a.ev_after && (e = hipEventRecord(a.ev_after, s)) != hipSuccess) return e;
    if (!plan.partial) return hipSuccess;
    return heads ? launch_project_finish(a, s) : launch_out_finish(a, s);
}

}  // namespace kva
