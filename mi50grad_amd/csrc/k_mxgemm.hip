// The projections by 4-bit weights (gfx950): microscaled rows of activations
// in 8 or 4 bits against packed 4-bit weight rows,
//   Y[t][n] = sum_k X[t][k] W[n][k],
// on v_mfma_scale_f32_32x32x64_f8f6f4 with weight rows as A and tokens as B:
// the products of a block of 32 are taken exactly, times both scales, and
// summed in fp32.  Lane l holds of A row l % 32's block l / 32 of a step of 64
// (16 bytes), of an 8-bit B token l % 32's bytes 16 (l / 32) .. +15 of either
// block (the instruction's order for 8 bits), of a 4-bit B its block l / 32,
// and of both one scale byte, of block l / 32; the result's register 4 q + j
// is token l % 32's row 8 q + 4 (l / 32) + j.
//
// Up to 32 tokens are bound by the weights, 17 bytes of each 32 values: 39 MB at
// 5120 -> 14336 (a read of memory takes 6.6 us).  mx_stream_kernel takes 8.8 us
// for one token and 10.5 to 12 for 32 of 8 bits, and 6.3 and 8.3 at 6144 -> 5120
// (17 MB, 3.0 us), where 160 workgroups do not fill the chip.  Each workgroup
// reads all of X, 32 tokens of 8 bits as many bytes as the weights; and of the 82
// lines of 128 bytes that a unit of one row tile touches, 32 are for a token's
// four bytes of scales each.
//
// More tokens are bound by the matrix units, or rather by what clock the card's
// power leaves them.  2048 tokens by mx_gemm_kernel, in us (and PFLOP/s), and a
// library's plain product of the same types with fp16 outputs, on one card (the
// first line takes 134 and 109 on a slower one):
//   5120 -> 14336, norm, RoPE and append   8 bits 127 (2.4)   4 bits 105 (2.9)
//     plain product                               124                117
//   6144 -> 5120 and a residual            8 bits  52 (2.5)   4 bits  51
//     plain product                                62                 67
// A tile of 256 x 256 starts in 2.3 us (its first stages) and ends in 7, or 13
// as a head; between, its loads, LDS reads and products are interleaved step by
// step, so that none of them waits in a row for the others.  Between 33 and some
// 500 tokens the tiles do not fill the chip: 181 tokens are 168 tiles of 64 x 256
// for 256 CUs and take 19 to 20 us, some 12 for 20 times 256 values and 7 to start
// and end as a head, where the products spread over the chip would take 10.
#include <algorithm>
#include <iterator>
#include <type_traits>
#include <utility>

#include "k_mx.h"
#include "k_normrope.h"
#include "kva_internal.h"

namespace kva {
namespace {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));

template <int BITS, int WSEL, int XSEL>
__device__ __forceinline__ float16_t mx_mfma(uint4 w, const uint4 (&x)[BITS == 8 ? 2 : 1], float16_t c, uint32_t ws,
                                             uint32_t xs) {
    const int8v_t wv = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
    int8v_t xv = {static_cast<int>(x[0].x), static_cast<int>(x[0].y), static_cast<int>(x[0].z), static_cast<int>(x[0].w), 0, 0, 0, 0};
    if constexpr (BITS == 8) {
        xv[4] = static_cast<int>(x[1].x);
        xv[5] = static_cast<int>(x[1].y);
        xv[6] = static_cast<int>(x[1].z);
        xv[7] = static_cast<int>(x[1].w);
    }
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, c, 4, BITS == 8 ? 0 : 4, WSEL, static_cast<int>(ws),
                                                           XSEL, static_cast<int>(xs));
}

__device__ __forceinline__ uint4 rsrc_b128(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0);
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// A pointer that every lane holds alike, in scalar registers (a buffer's base).
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const auto v = reinterpret_cast<uintptr_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return reinterpret_cast<const uint8_t *>(static_cast<uintptr_t>(hi) << 32 | lo);
}

// A barrier that waits for LDS alone: __syncthreads() would also wait until
// every store has arrived, some 2 us.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    wait_vm_lds<63>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ float16_t zero16() {
    return float16_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

// The packed weight that row tile `rt` of the stacked rows lies in, and its
// place there.
struct MxTileAt {
    const uint8_t *codes, *scales;  // of the tile
};
__device__ __forceinline__ MxTileAt mx_tile_at(const ProjectArgs &a, const MxProduct &m, int rt) {
    const int rta = a.n_a / kMxWeightTile;
    const bool first = rt < rta || a.n_b == 0;
    const uint8_t *w = first ? m.w_a : m.w_b;
    const int64_t t = first ? rt : rt - rta;
    const int64_t tiles = ((first ? a.n_a : a.n_b) + kMxWeightTile - 1) / kMxWeightTile;
    return {w + t * 16 * a.hidden, w + tiles * 16 * a.hidden + t * a.hidden};
}

// On the lambdas of the main loop: one that stays a call puts the registers
// that it refers to into memory.
#define KVA_INLINE __attribute__((always_inline))

template <int V>
using Int = std::integral_constant<int, V>;

// f(Int<FROM>), ..., f(Int<TO - 1>).
template <int FROM, class F, int... I>
__device__ __forceinline__ void each_of(const F &f, std::integer_sequence<int, I...>) {
    (f(Int<FROM + I>{}), ...);
}
template <int FROM, int TO, class F>
__device__ __forceinline__ void each(const F &f) {
    each_of<FROM>(f, std::make_integer_sequence<int, TO - FROM>{});
}

// The granule swizzle of a row of 128 bytes: the 16 rows that 16 lanes read
// at one granule fall in distinct 16-byte bank groups.
__device__ __forceinline__ int mx_swizzle(int r) { return ((r >> 1) ^ ((r & 1) << 2)) & 7; }

// ---- up to 32 tokens ---------------------------------------------------------

constexpr int kMxStreamWaves = 8;

// A unit of the streaming form: 128 values of k of RT row tiles and of TOK
// tokens, with their scales, in one of the wave's own S slots.
template <int BITS_, int RT_, int TOK_>
struct MxUnit {
    static constexpr int BITS = BITS_, RT = RT_, TOK = TOK_;
    static constexpr int kXRow = 16 * BITS;           // bytes of a token
    static constexpr int kX = TOK * kXRow < 1024 ? 1024 : TOK * kXRow, kW = RT * 2048, kXs = 256, kWs = RT * 256;
    static constexpr int kSlot = kX + kW + kXs + kWs;
    static constexpr int kLoads = kX / 1024 + kW / 1024 + 1 + RT;
    static constexpr int S = 20 * 1024 / kSlot;       // the LDS shared by eight waves
    static_assert(S >= 2 && kLoads * (S - 1) < 64, "one unit at least on its way, vmcnt is six bits");
    static_assert(kMxStreamWaves * S * kSlot >= kMxStreamWaves * RT * 4096, "the waves' sums fit");
};

// A workgroup takes RT row tiles over the whole of hidden, a run of units per
// wave, through loads that write the wave's own slots of LDS: no wave waits for
// another, a token's row comes in whole lines (operands straight from memory
// touch a line per token and instruction, four times as many: 32 tokens of 6144
// -> 5120 took 12.6 us).  The waves' sums meet in LDS.  No k is split among
// workgroups, so with OUT the result is finished here; else fp32 rows go to a
// finish kernel.
template <int BITS, int RT, int TOK, bool OUT>
__global__ __launch_bounds__(64 * kMxStreamWaves) void mx_stream_kernel(ProjectArgs a, MxProduct m) {
    using U = MxUnit<BITS, RT, TOK>;
    __shared__ __attribute__((aligned(16))) uint8_t ring[kMxStreamWaves][U::S * U::kSlot];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int N = a.n_a + a.n_b, K = a.hidden;
    const int rt0 = blockIdx.x * RT, n_rt = (N + kMxWeightTile - 1) / kMxWeightTile;
    const int units = K / 128;
    const int u0 = wave * units / kMxStreamWaves, n = (wave + 1) * units / kMxStreamWaves - u0;
    const uint8_t *w_at[RT], *ws_at[RT];
    uint32_t w_size[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const MxTileAt at = mx_tile_at(a, m, min(rt0 + i, n_rt - 1));
        w_at[i] = uniform(at.codes);
        ws_at[i] = uniform(at.scales);
        w_size[i] = __builtin_amdgcn_readfirstlane(rt0 + i < n_rt ? static_cast<uint32_t>(K) : 0u);
    }
    const uint32_t x_row = static_cast<uint32_t>(K) * BITS / 8, s_row = static_cast<uint32_t>(K) / 32;
    // Loads of X: 1 KB of whole rows, granules swizzled so that the 16 rows that
    // 16 lanes read at one fall in distinct banks.
    constexpr int kLanes = U::kXRow / 16, kRows = 64 / kLanes;  // lanes of a row, rows of a load
    auto swizzle = [](int r) { return BITS == 8 ? mx_swizzle(r) : (r >> 2) & 3; };
    uint32_t xoff[U::kX / 1024];
#pragma unroll
    for (int j = 0; j < U::kX / 1024; ++j) {
        const int row = kRows * j + lane / kLanes;
        xoff[j] = row * x_row + 16 * ((lane % kLanes) ^ swizzle(row));
    }
    // A column past TOK is a copy of one that is not, and not stored.
    const int tok = col % TOK;
    const uint32_t xs_off = tok * s_row, lds0 = lds_addr(ring[wave]);
    // Units past the wave's last go through empty buffers, so that every wait counts alike.
    auto issue = [&](int i) {
        const bool on = i < n;
        const uint32_t u = on ? static_cast<uint32_t>(u0 + i) : 0u;
        const uint32_t st = lds0 + i % U::S * U::kSlot;
        const uint32_t toks = on ? static_cast<uint32_t>(a.n_tok) : 0u;
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const auto rw = ro_rsrc(w_at[j], on ? w_size[j] * 16 : 0u), rs = ro_rsrc(ws_at[j], on ? w_size[j] + 0u : 0u);
            load_to_lds_at(rw, st + U::kX + 2048 * j, 16 * lane, u * 2048);
            load_to_lds_at(rw, st + U::kX + 2048 * j + 1024, 16 * lane + 1024, u * 2048);
            word_to_lds_at(rs, st + U::kX + U::kW + U::kXs + 256 * j, 4 * lane, u / 2 * 256);
        }
        const auto rx = ro_rsrc(m.x, toks * x_row), rxs = ro_rsrc(m.x_scales, toks * s_row);
#pragma unroll
        for (int j = 0; j < U::kX / 1024; ++j) load_to_lds_at(rx, st + 1024 * j, xoff[j], u * U::kXRow);
        word_to_lds_at(rxs, st + U::kX + U::kW, xs_off, u * 4);
    };
    float16_t acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = zero16();
    for (int i = 0; i < U::S; ++i) issue(i);
    for (int i = 0; i < n; ++i) {
        wait_vm<U::kLoads *(U::S - 1)>();
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *st = ring[wave] + i % U::S * U::kSlot;
        constexpr int XV = BITS == 8 ? 2 : 1;
        uint4 x[2][XV], w[2][RT];
        uint32_t ws[RT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int v = 0; v < XV; ++v) {
                const int g = BITS == 8 ? 4 * s + 2 * v + half : 2 * s + half;
                x[s][v] = *reinterpret_cast<const uint4 *>(st + tok * U::kXRow + 16 * (g ^ swizzle(tok)));
            }
#pragma unroll
            for (int j = 0; j < RT; ++j)
                w[s][j] = *reinterpret_cast<const uint4 *>(st + U::kX + 2048 * j + 1024 * s + 16 * lane);
        }
        const uint32_t xs = *reinterpret_cast<const uint32_t *>(st + U::kX + U::kW + 4 * lane) >> (8 * half);
#pragma unroll
        for (int j = 0; j < RT; ++j)
            ws[j] = *reinterpret_cast<const uint32_t *>(st + U::kX + U::kW + U::kXs + 256 * j + 4 * lane) >> (16 * ((u0 + i) & 1));
        // The slot has been read before it is loaded again.
        wait_vm_lds<63>();
        __builtin_amdgcn_sched_barrier(0);
        issue(i + U::S);
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            acc[j] = mx_mfma<BITS, 0, 0>(w[0][j], x[0], acc[j], ws[j], xs);
            acc[j] = mx_mfma<BITS, 1, 2>(w[1][j], x[1], acc[j], ws[j], xs);
        }
    }
    // Every load (the empty ones too) has landed before the LDS is handed on.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    float4_t *red = reinterpret_cast<float4_t *>(ring);  // [wave][RT][4][64]
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            red[((wave * RT + i) * 4 + q) * 64 + lane] =
                float4_t{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
    __syncthreads();
    // Eight threads finish a token's 32 rows of a tile.
    for (int f = threadIdx.x; f < RT * 256; f += 64 * kMxStreamWaves) {
        const int i = f >> 8, t = (f >> 3) & 31, rq = f & 7;
        if (t >= a.n_tok) continue;
        const int row = 32 * (rt0 + i) + 4 * rq;
        if (row >= N) continue;
        const size_t at = static_cast<size_t>(t) * N + row;
        uint2 r = make_uint2(0, 0);
        if (OUT && a.residual) r = ld8(a.residual + at);
        const int from = t + 32 * (rq & 1);
        float4_t sum = red[(i * 4 + (rq >> 1)) * 64 + from];
#pragma unroll
        for (int w = 1; w < kMxStreamWaves; ++w) sum += red[((w * RT + i) * 4 + (rq >> 1)) * 64 + from];
        if constexpr (OUT) {
            sum += float4_t{lo_f(r.x), hi_f(r.x), lo_f(r.y), hi_f(r.y)};
            *reinterpret_cast<uint2 *>(a.y_out + at) = make_uint2(pack_h2(sum[0], sum[1]), pack_h2(sum[2], sum[3]));
        } else {
            *reinterpret_cast<float4_t *>(a.part + at) = sum;
        }
    }
}

// ---- tiles -------------------------------------------------------------------

enum MxEpilogue {
    kMxHead,  // a tile is a head's rows: norm + RoPE, outputs, cache rows
    kMxOut,   // out = fp16(sum + residual)
    kMxPart,  // fp32 partials [split][token][row] for a finish kernel
};

// A tile of BM tokens x BN weight rows over WM x WN waves and S LDS stages of
// KC values of k.
template <int BITS_, int BM_, int BN_, int WM_, int WN_, int S_>
struct MxTile {
    static constexpr int BITS = BITS_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
    static constexpr int kWaves = WM * WN;
    static constexpr int KC = BITS == 8 ? 128 : 256;  // a row's 128-byte line
    static constexpr int SPC = KC / 64;               // steps of a stage
    static constexpr int kTM = BM / WM / 32, kTN = BN / WN / 32;  // MFMA tiles of a wave
    static constexpr int XV = BITS == 8 ? 2 : 1;      // 16-byte pieces of a token's step
    static constexpr int kStageX = BM * 128, kStageW = BN / 32 * SPC * 1024, kStage = kStageX + kStageW;
    static constexpr int kPlanes = KC / 128;          // dwords of a token's scales in a chunk
    static constexpr int kParts = 512 / KC;           // chunks that share a load of scales
    static constexpr int kSmall = (BM + BN) / 64;     // loads of 1 KB of scales, for 512 values of k
    static constexpr int kLoadsX = kStageX / 1024 / kWaves, kLoadsW = kStageW / 1024 / kWaves;
    static constexpr int kLoadsS = (kSmall + kWaves - 1) / kWaves;
    // With room for what the waves load only to keep their count.
    static constexpr int kScales = 1024 * (kSmall + (kSmall % kWaves ? 1 : 0));
    // Scales of 512 arrive while those of earlier chunks are still read.
    static constexpr int kScaleBufs = (S - 2) / kParts + 2;
    static constexpr int kRing = S * kStage + kScaleBufs * kScales;
    // Loads of a wave for chunk `part` of its 512, and for chunks [from, to).
    static constexpr int loads(int part) { return kLoadsX + kLoadsW + (part % kParts == 0 ? kLoadsS : 0); }
    static constexpr int loads(int from, int to) { return from < to ? loads(from) + loads(from + 1, to) : 0; }
    // Of a chunk's loads, those of its first `steps` steps.
    static constexpr int share(int part, int steps) { return loads(part) * steps / SPC; }
    static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && BM % 64 == 0 && BN % 64 == 0,
                  "whole MFMA tiles and loads");
    static_assert(kLoadsX * kWaves * 1024 == kStageX && kLoadsW * kWaves * 1024 == kStageW, "whole loads per wave");
    static_assert(S >= 2 && loads(0, S) < 64, "vmcnt is six bits");
    static_assert(kRing <= 160 * 1024, "the ring fits the LDS");
    static_assert(BM <= 64 * kWaves, "a thread a token");
};

// Workgroup i runs on XCD i % 8: deal each XCD a contiguous run of n tiles.
__device__ __forceinline__ int mx_deal(int i, int n) {
    const int xcd = i & 7, q8 = n >> 3, r8 = n & 7;
    return xcd * q8 + min(xcd, r8) + (i >> 3);
}

template <class T, int EPI>
__global__ __launch_bounds__(64 * T::kWaves) void mx_gemm_kernel(ProjectArgs a, MxProduct m) {
    constexpr int kTM = T::kTM, kTN = T::kTN, SPC = T::SPC, BITS = T::BITS, XV = T::XV;
    __shared__ __attribute__((aligned(16))) uint8_t ring[T::kRing];
    const int N = a.n_a + a.n_b, K = a.hidden;
    const int n_rt = (N + T::BN - 1) / T::BN, n_mt = (a.n_tok + T::BM - 1) / T::BM;
    const int splits = EPI == kMxPart ? a.splits : 1;
    // With `by_kind` the first half of the workgroups takes Q and K heads, the
    // second gate and V.
    const bool by_kind = EPI == kMxHead && m.by_kind;
    const int n_wg = n_rt * splits * n_mt / (by_kind ? 2 : 1), wg = blockIdx.x;
    const bool second = by_kind && wg >= n_wg;
    const int tau = mx_deal(second ? wg - n_wg : wg, n_wg);
    // Token tiles fastest, then row tiles, then splits.
    const int ws_at = __builtin_amdgcn_readfirstlane(tau / n_mt);
    const int mt = __builtin_amdgcn_readfirstlane(tau - ws_at * n_mt);
    const int split = EPI == kMxPart ? __builtin_amdgcn_readfirstlane(ws_at / n_rt) : 0;
    const int H = a.num_heads, hkv = a.num_kv_heads;
    const int rt = !by_kind      ? ws_at - split * n_rt
                   : ws_at < H ? ws_at + (second ? H : 0)
                                 : ws_at + H + (second ? hkv : 0);
    const int t0 = mt * T::BM, n0 = rt * T::BN;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;

    // The facts of the tile's tokens (RoPE position, slot, page), a thread a
    // token: requested first, used last.
    int3 fact = make_int3(0, 0, 0);
    if (EPI == kMxHead && threadIdx.x < T::BM) {
        const int t = min(t0 + static_cast<int>(threadIdx.x), a.n_tok - 1);
        fact.x = a.tok_pos[t];
        fact.y = a.tok_slot[t];
        fact.z = a.table[static_cast<size_t>(a.tok_seq[t]) * a.table_stride + (fact.y >> 4)];
    }

    // The operands as buffers: rows past the last token and tiles past the
    // last weight row read as zeros.
    const uint32_t x_row = static_cast<uint32_t>(K) * BITS / 8, s_row = static_cast<uint32_t>(K) / 32;
    const uint32_t toks = static_cast<uint32_t>(max(0, min(T::BM, a.n_tok - t0)));
    const MxTileAt at = mx_tile_at(a, m, n0 / 32);
    const uint32_t tiles = static_cast<uint32_t>((min(T::BN, N - n0) + 31) / 32);
    const uint8_t *const x_at = uniform(m.x + static_cast<size_t>(t0) * x_row), *const w_at = uniform(at.codes);
    const uint8_t *const xs_at = m.x_scales + static_cast<size_t>(t0) * s_row;
    const uint32_t x_size = __builtin_amdgcn_readfirstlane(toks * x_row);
    const uint32_t w_size = __builtin_amdgcn_readfirstlane(tiles * 16u * K);
    const uint32_t lds0 = lds_addr(ring);
    // This split's chunks: slices of hidden are whole 512s.
    const int n512 = K / 512;
    const int cb = EPI == kMxPart ? __builtin_amdgcn_readfirstlane(split * n512 / splits) * T::kParts : 0;
    const int nc =
        (EPI == kMxPart ? __builtin_amdgcn_readfirstlane((split + 1) * n512 / splits) : n512) * T::kParts - cb;

    uint32_t xoff[T::kLoadsX], woff[T::kLoadsW];
#pragma unroll
    for (int j = 0; j < T::kLoadsX; ++j) {
        const int row = 8 * (T::kWaves * j + wv) + (lane >> 3);
        xoff[j] = row * x_row + 16 * ((lane & 7) ^ mx_swizzle(row));
    }
#pragma unroll
    for (int j = 0; j < T::kLoadsW; ++j) {
        const int q = T::kWaves * j + wv;
        woff[j] = (q / SPC) * 16u * K + (q % SPC) * 1024u + 16 * lane;
    }
    // A load of scales, for 512 values of k: 16 bytes of 64 tokens, or 512 of
    // two row tiles, or none, where a wave loads only to keep its count.  (Four
    // bytes of a token per chunk of 128 would bring a line each time.  At 2048 x
    // 14336 x 5120 that took the same: 145.7 us against 145.2.)
    const uint8_t *sm_at[T::kLoadsS];
    uint32_t sm_size[T::kLoadsS], sm_step[T::kLoadsS], sm_off[T::kLoadsS];
#pragma unroll
    for (int j = 0; j < T::kLoadsS; ++j) {
        const int q = T::kWaves * j + wv, qw = q - T::BM / 64;
        const bool of_x = qw < 0;
        sm_at[j] = uniform(of_x ? xs_at : at.scales);
        sm_size[j] = __builtin_amdgcn_readfirstlane(of_x            ? toks * s_row
                                                    : q < T::kSmall ? tiles * static_cast<uint32_t>(K)
                                                                    : 0u);
        // An empty buffer is read at 0 alone: a range check may subtract the scalar
        // offset from the size.
        sm_step[j] = of_x ? 16 : q < T::kSmall ? 512 : 0;
        sm_off[j] = of_x ? (64 * q + lane) * s_row : (2 * qw + half) * static_cast<uint32_t>(K) + 16 * col;
    }
    // Piece j of the loads of chunk c into the stage at `st`.  A chunk past the
    // end goes through empty buffers: the same loads, no memory access, so
    // every wave's load counter advances alike.
    auto load = [&](auto piece, int c, uint32_t st) KVA_INLINE {
        constexpr int j = decltype(piece)::value;
        const bool on = c < nc;
        const uint32_t k = on ? static_cast<uint32_t>(cb + c) : 0u;
        if constexpr (j < T::kLoadsX) {
            load_to_lds_at(ro_rsrc(x_at, on ? x_size + 0u : 0u), st + 1024 * (T::kWaves * j + wv), xoff[j], k * 128);
        } else if constexpr (j < T::kLoadsX + T::kLoadsW) {
            constexpr int i = j - T::kLoadsX;
            load_to_lds_at(ro_rsrc(w_at, on ? w_size + 0u : 0u), st + T::kStageX + 1024 * (T::kWaves * i + wv),
                           woff[i], k * (SPC * 1024));
        } else {
            constexpr int i = j - T::kLoadsX - T::kLoadsW;
            const uint32_t dst = T::S * T::kStage + c / T::kParts % T::kScaleBufs * T::kScales;
            load_to_lds_at(ro_rsrc(sm_at[i], on ? sm_size[i] + 0u : 0u),
                           lds0 + dst + 1024 * min(T::kWaves * i + wv, T::kSmall), sm_off[i],
                           __builtin_amdgcn_readfirstlane(k / T::kParts * sm_step[i]));
        }
    };

    const int wm = wv / T::WN, wn = wv % T::WN;
    float16_t acc[kTM][kTN];
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTN; ++j) acc[i][j] = zero16();

    // Operands are read from LDS a step ahead, and a chunk's scales with its
    // first step's: of each token tile a dword per 128 k (its bytes 0 and 2,
    // shifted by this lane's half), of each row tile the bytes of four steps.
    constexpr int kReads = kTN + kTM * XV, kScaleReads = kTM * T::kPlanes + kTN;
    struct Step {
        uint4 x[kTM][XV], w[kTN];
    };
    struct Scales {
        uint32_t x[kTM][T::kPlanes], w[kTN];
    };
    auto read = [&](auto piece, Step &o, const uint8_t *st, int s) KVA_INLINE {
        constexpr int p = decltype(piece)::value;
        if constexpr (p < kTN) {
            o.w[p] = *reinterpret_cast<const uint4 *>(st + T::kStageX + ((wn * kTN + p) * SPC + s) * 1024 + 16 * lane);
        } else {
            constexpr int i = (p - kTN) / XV, v = (p - kTN) % XV;
            const int row = (wm * kTM + i) * 32 + col;
            const int g = BITS == 8 ? 4 * s + 2 * v + half : 2 * s + half;
            o.x[i][v] = *reinterpret_cast<const uint4 *>(st + row * 128 + 16 * (g ^ mx_swizzle(row)));
        }
    };
    // Piece p of the scales of chunk `part` of its 512, which are at `at`.
    auto read_scale = [&](auto piece, auto part, Scales &o, const uint8_t *from) KVA_INLINE {
        constexpr int p = decltype(piece)::value, k = decltype(part)::value * T::KC;
        if constexpr (p < kTN) {
            o.w[p] = *reinterpret_cast<const uint32_t *>(from + T::BM * 16 + (wn * kTN + p) * 512 + k / 256 * 256 + 4 * lane);
        } else {
            constexpr int i = (p - kTN) / T::kPlanes, pl = (p - kTN) % T::kPlanes;
            o.x[i][pl] = *reinterpret_cast<const uint32_t *>(from + ((wm * kTM + i) * 32 + col) * 16 + 4 * (k / 128 + pl));
        }
    };
    // A step's products, with hook(k) after the k-th: what the wave issues
    // there runs under the products instead of between two steps.
    constexpr int kProducts = kTM * kTN;
    auto multiply = [&](auto s, auto ws, const Step &o, const Scales &sc, const auto &hook) KVA_INLINE {
        constexpr int kS = decltype(s)::value, kWs = decltype(ws)::value;
        each<0, kProducts>([&](auto k) KVA_INLINE {
            constexpr int i = decltype(k)::value / kTN, j = decltype(k)::value % kTN;
            acc[i][j] = mx_mfma<BITS, kWs, 2 * (kS & 1)>(o.w[j], o.x[i], acc[i][j], sc.w[j], sc.x[i][kS >> 1]);
            hook(k);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // What comes after product k of n pieces spread over the first `over`.
    auto spread = [](auto k, auto n, auto over, const auto &piece) KVA_INLINE {
        constexpr int kK = decltype(k)::value, kN = decltype(n)::value, kOver = decltype(over)::value;
        if constexpr (kK < kOver) each<kN * kK / kOver, kN * (kK + 1) / kOver>(piece);
    };
    // Reads come early, so that the last has arrived when its step begins.
    using Early = Int<kProducts - kProducts / 4>;
    using Whole = Int<kProducts>;
    // Chunk c + S is loaded from c's last step on, when its stage is free, a
    // share of it in each step until the next chunk's last: piled up in one
    // step, four waves' loads hold up each other's products.
    each<0, T::S - 1>([&](auto c) KVA_INLINE {
        each<0, T::loads(decltype(c)::value)>([&](auto j) KVA_INLINE { load(j, c, lds0 + c * T::kStage); });
    });
    each<0, T::share(T::S - 1, 1)>([&](auto j) KVA_INLINE { load(j, T::S - 1, lds0 + (T::S - 1) * T::kStage); });
    wait_vm<T::loads(1, T::S - 1) + T::share(T::S - 1, 1)>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    Step o0, o1;
    Scales sc0, sc1;
    each<0, kReads>([&](auto p) KVA_INLINE { read(p, o0, ring, 0); });
    each<0, kScaleReads>([&](auto p) KVA_INLINE { read_scale(p, Int<0>{}, sc0, ring + T::S * T::kStage); });
    uint32_t before = (T::S - 1) * T::kStage, at0 = 0;  // the last chunk's stage and this one's
    // Chunk c, `part` of its 512.
    auto chunk = [&](auto part, int c, Scales &sc, Scales &sc_next) KVA_INLINE {
        constexpr int kPart = decltype(part)::value;
        const uint32_t at1 = at0 + T::kStage == T::S * T::kStage ? 0 : at0 + T::kStage;
        const uint8_t *st = ring + at0, *next = ring + at1;
        const uint8_t *next_scales = ring + T::S * T::kStage + (c + 1) / T::kParts % T::kScaleBufs * T::kScales;
        each<0, kTM>([&](auto i) KVA_INLINE { each<0, T::kPlanes>([&](auto p) KVA_INLINE { sc.x[i][p] >>= 8 * half; }); });
        auto one = [&](auto s, Step &now, Step &then) KVA_INLINE {
            constexpr int kS = decltype(s)::value;
            using Ws = Int<(kPart * SPC + kS) % 4>;
            if constexpr (kS + 1 < SPC) {
                multiply(s, Ws{}, now, sc, [&](auto k) KVA_INLINE {
                    spread(k, Int<kReads>{}, Early{}, [&](auto p) KVA_INLINE { read(p, then, st, kS + 1); });
                    constexpr int kPiece = T::share(kPart + T::S - 1, kS + 1), kEnd = T::share(kPart + T::S - 1, kS + 2);
                    spread(k, Int<kEnd - kPiece>{}, Whole{}, [&](auto j) KVA_INLINE {
                        load(Int<kPiece + decltype(j)::value>{}, c + T::S - 1, lds0 + before);
                    });
                });
            } else {
                // This wave has read all of chunk c, and chunk c + 1 has landed.
                wait_vm_lds<T::loads(kPart + 2, kPart + T::S)>();
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
                multiply(s, Ws{}, now, sc, [&](auto k) KVA_INLINE {
                    spread(k, Int<kReads + kScaleReads>{}, Early{}, [&](auto p) KVA_INLINE {
                        if constexpr (decltype(p)::value < kReads) read(p, then, next, 0);
                        else read_scale(Int<decltype(p)::value - kReads>{}, Int<(kPart + 1) % T::kParts>{}, sc_next, next_scales);
                    });
                    spread(k, Int<T::share(kPart + T::S, 1)>{}, Whole{},
                           [&](auto j) KVA_INLINE { load(j, c + T::S, lds0 + at0); });
                });
            }
        };
        one(Int<0>{}, o0, o1);
        one(Int<1>{}, o1, o0);
        if constexpr (SPC == 4) {
            one(Int<2>{}, o0, o1);
            one(Int<3>{}, o1, o0);
        }
        before = at0;
        at0 = at1;
    };
    for (int c = 0; c < nc; c += T::kParts) {
        chunk(Int<0>{}, c, sc0, sc1);
        chunk(Int<1>{}, c + 1, sc1, sc0);
        if constexpr (T::kParts == 4) {
            chunk(Int<2>{}, c + 2, sc0, sc1);
            chunk(Int<3>{}, c + 3, sc1, sc0);
        }
    }
    // Every load (the dummy ones past the end too) has landed before the LDS
    // is handed on.
    __builtin_amdgcn_s_waitcnt(0);

    // The sums leave through LDS, 32 tokens of every wave row at a time, so that
    // whole lines are stored (a lane's four rows of its token in place took 7 to
    // 11 us a tile, 16 bytes of each line at once): LPR lanes a token's row,
    // eight rows of the weight each.
    constexpr int kRow = T::BN + 4;  // floats of a token's strip row, padded against bank conflicts
    constexpr int kStripToks = 32 * T::WM, kStrip = kStripToks * kRow * 4;
    constexpr int LPR = T::BN / 8, kThreads = 64 * T::kWaves, kPer = kStripToks * LPR / kThreads;
    static_assert(kPer * kThreads == kStripToks * LPR, "as many pieces for every thread");
    static_assert(EPI != kMxHead || T::BN == kHeadDim, "a head tile holds whole heads");
    static_assert(kStrip + 3 * 4 * T::BM <= T::kRing, "a strip of tokens and the tokens' facts fit the ring");
    float *strip = reinterpret_cast<float *>(ring);
    int32_t *facts = reinterpret_cast<int32_t *>(ring + kStrip);
    const int l = threadIdx.x % LPR;  // of a head's row, where it is the same for every piece
    __syncthreads();
    if constexpr (EPI == kMxHead) {
        if (threadIdx.x < T::BM) {
            facts[threadIdx.x] = fact.x;
            facts[T::BM + threadIdx.x] = fact.y;
            facts[2 * T::BM + threadIdx.x] = fact.z;
        }
        __syncthreads();
    }
    const int head = rt;
    const bool is_q = head < H, is_gate = !is_q && head < 2 * H;
    const int kv = head - 2 * H;  // K heads 0..hkv-1, then V heads
    const bool rot = EPI == kMxHead && (is_q || (!is_gate && kv < hkv));
    const uint4 wnorm = rot ? ld16((is_q ? a.q_w : a.k_w) + 8 * l) : make_uint4(0, 0, 0, 0);
    const int cl = a.half_rot > 0 ? min(l, a.half_rot / 4 - 1) : 0;
    // Rows are stored, and residuals read, through buffers over the tile's
    // tokens: those past the last fall out of range without a branch, and so
    // do columns past the last row (far).  A null output is an empty buffer.
    constexpr uint32_t far = 0x80000000u;
    const void *to = EPI == kMxPart  ? static_cast<const void *>(a.part + (static_cast<size_t>(split) * a.n_tok + t0) * N)
                     : EPI == kMxOut ? a.y_out + static_cast<size_t>(t0) * N
                     : is_q          ? a.q_out + static_cast<size_t>(t0) * H * kHeadDim
                     : is_gate       ? a.gate_out + (a.gate_out ? static_cast<size_t>(t0) * H * kHeadDim : 0)
                                     : a.kv_out + (a.kv_out ? static_cast<size_t>(t0) * 2 * hkv * kHeadDim : 0);
    const uint32_t line = EPI == kMxPart  ? 4u * N
                          : EPI == kMxOut ? 2u * N
                                          : 2u * kHeadDim * (is_q || is_gate ? H : 2 * hkv);
    const uint32_t head_col = 2u * kHeadDim * (is_q ? head : is_gate ? head - H : kv) + 16u * l;
    const uint8_t *to_at = uniform(static_cast<const uint8_t *>(to));
    const auto rto = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(to_at), 0, __builtin_amdgcn_readfirstlane(to_at ? toks * line : 0u), 0x00020000);
    const uint8_t *res_at = uniform(reinterpret_cast<const uint8_t *>(a.residual ? a.residual + static_cast<size_t>(t0) * N : nullptr));
    const auto rres = ro_rsrc(res_at, __builtin_amdgcn_readfirstlane(EPI == kMxOut && res_at ? toks * line : 0u));
    // This thread's piece j of part i of the tile: its row of the strip, its
    // token, and its place from there.
    auto strip_row = [&](int j) KVA_INLINE { return static_cast<int>(threadIdx.x + kThreads * j) / LPR; };
    auto token = [&](int i, int j) KVA_INLINE {
        const int sr = strip_row(j);
        return ((sr >> 5) * kTM + i) * 32 + (sr & 31);
    };
    auto lane_of = [&](int j) KVA_INLINE { return static_cast<int>(threadIdx.x + kThreads * j) % LPR; };
    auto at_col = [&](int j) KVA_INLINE {
        const int n = n0 + 8 * lane_of(j);  // its first row of the weight
        return EPI == kMxHead ? head_col : n < N ? (EPI == kMxPart ? 4u : 2u) * n : far;
    };
    // What finishing part i reads, requested a part ahead: before the stores
    // that would be waited for with it.
    struct Ahead {
        uint4 res[EPI == kMxOut ? kPer : 1];
        uint2 c[EPI == kMxHead ? kPer : 1], s[EPI == kMxHead ? kPer : 1];
    };
    auto request = [&](Ahead &o, int i) KVA_INLINE {
        if constexpr (EPI == kMxOut) {
            each<0, kPer>([&](auto j) KVA_INLINE { o.res[j] = rsrc_b128(rres, token(i, j) * line + at_col(j), 0); });
        } else if constexpr (EPI == kMxHead) {
            each<0, kPer>([&](auto j) KVA_INLINE {
                // Tokens past the last carry its position: inside the tables.
                const size_t off = static_cast<size_t>(facts[token(i, j)]) * a.half_rot + 4 * cl;
                const uint16_t *w = is_q ? a.q_w : a.k_w;  // without a rotary part: in bounds, not used
                o.c[j] = ld8(a.half_rot > 0 ? a.cos_tab + off : w);
                o.s[j] = ld8(a.half_rot > 0 ? a.sin_tab + off : w);
            });
        }
    };
    auto store = [&](uint4 v, uint32_t off) KVA_INLINE {
        typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b128(u4_t{v.x, v.y, v.z, v.w}, rto, off, 0, 0);
    };
    Ahead now, then;
    request(now, 0);
#pragma unroll 1
    for (int i = 0; i < kTM; ++i) {
        each<0, kTM>([&](auto part) KVA_INLINE {
            if (i != part) return;
            each<0, kTN>([&](auto j) KVA_INLINE {
                each<0, 4>([&](auto q) KVA_INLINE {
                    *reinterpret_cast<float4_t *>(strip + (wm * 32 + col) * kRow + (wn * kTN + j) * 32 + 8 * q + 4 * half) =
                        float4_t{acc[part][j][4 * q], acc[part][j][4 * q + 1], acc[part][j][4 * q + 2], acc[part][j][4 * q + 3]};
                });
            });
        });
        lds_barrier();
        request(then, min(i + 1, kTM - 1));
        if constexpr (EPI == kMxHead) {
            // In fp32 up to here: Q and K are rounded once, after norm and RoPE.
            // All rows are worked out before the first is stored, so that their
            // sums across lanes run side by side.
            uint4 y[kPer], o[kPer];
            auto row = [&](int j, float (&x)[8]) KVA_INLINE {
                const float *from = strip + strip_row(j) * kRow + 8 * l;
                const float4_t lo = *reinterpret_cast<const float4_t *>(from), hi = *reinterpret_cast<const float4_t *>(from + 4);
                x[0] = lo[0], x[1] = lo[1], x[2] = lo[2], x[3] = lo[3], x[4] = hi[0], x[5] = hi[1], x[6] = hi[2], x[7] = hi[3];
                return make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
            };
            if (rot) {
                // A square root and a division take some 25 instructions: lane l
                // takes row l % kPer's and hands them on (each lane all of its rows': 127.7
                // us for 126.8 at 2048 tokens of 5120 -> 14336, in 4 bits 107.2 for 105.4).
                static_assert((kPer & (kPer - 1)) == 0 && kPer <= LPR, "a lane a row");
                float mine = 0.f;
                each<0, kPer>([&](auto j) KVA_INLINE {
                    float x[8];
                    y[j] = row(j, x);
                    const float sum = sum32_moves(sum_squares(x));
                    mine = (l & (kPer - 1)) == j ? sum : mine;
                });
                const int inv = __builtin_bit_cast(int, inv_rms<32>(mine, a.eps));
                each<0, kPer>([&](auto j) KVA_INLINE {
                    float x[8];
                    row(j, x);
                    constexpr int kLane = decltype(j)::value << 5;  // of 32: lane j's
                    const float by = __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(inv, kLane));
                    o[j] = norm_rope_by(x, NormRopeIn{wnorm, now.c[j], now.s[j]}, a.half_rot, by, l);
                });
            } else {
                each<0, kPer>([&](auto j) KVA_INLINE {
                    float x[8];
                    y[j] = o[j] = row(j, x);
                });
            }
            if (is_q) {
                each<0, kPer>([&](auto j) KVA_INLINE { store(o[j], token(i, j) * line + at_col(j)); });
            } else {
                each<0, kPer>([&](auto j) KVA_INLINE { store(y[j], token(i, j) * line + at_col(j)); });
            }
            if (kv >= 0) {
                uint16_t *const pool = kv < hkv ? a.k_pool + kv * kHeadDim : a.v_pool + (kv - hkv) * kHeadDim;
                each<0, kPer>([&](auto j) KVA_INLINE {
                    const int r = token(i, j);
                    const size_t at_row = static_cast<size_t>(facts[2 * T::BM + r]) * kBlockTokens + (facts[T::BM + r] & 15);
                    if (t0 + r < a.n_tok) st16(pool + at_row * hkv * kHeadDim + 8 * l, o[j]);
                });
            }
        } else {
            each<0, kPer>([&](auto j) KVA_INLINE {
                const uint32_t off = token(i, j) * line + at_col(j);
                const float *from = strip + strip_row(j) * kRow + 8 * lane_of(j);
                float4_t lo = *reinterpret_cast<const float4_t *>(from), hi = *reinterpret_cast<const float4_t *>(from + 4);
                if constexpr (EPI == kMxPart) {
                    store(__builtin_bit_cast(uint4, lo), off);
                    store(__builtin_bit_cast(uint4, hi), off + 16);
                } else {
                    // A lane reads its residual before it writes the same
                    // bytes, so out may be the residual.
                    const uint4 z = now.res[j];
                    lo += float4_t{lo_f(z.x), hi_f(z.x), lo_f(z.y), hi_f(z.y)};
                    hi += float4_t{lo_f(z.z), hi_f(z.z), lo_f(z.w), hi_f(z.w)};
                    store(make_uint4(pack_h2(lo[0], lo[1]), pack_h2(lo[2], lo[3]), pack_h2(hi[0], hi[1]), pack_h2(hi[2], hi[3])),
                          off);
                }
            });
        }
        lds_barrier();  // the strip is read before the next tokens overwrite it
        now = then;
    }
}

template <class T, int EPI>
hipError_t launch_mx_gemm(const ProjectArgs &a, const MxProduct &m, hipStream_t s) {
    const int n_rt = (a.n_a + a.n_b + T::BN - 1) / T::BN, n_mt = (a.n_tok + T::BM - 1) / T::BM;
    const int splits = EPI == kMxPart ? a.splits : 1;
    hipLaunchKernelGGL((mx_gemm_kernel<T, EPI>), dim3(n_rt * splits * n_mt), dim3(64 * T::kWaves), 0, s, a, m);
    return hipGetLastError();
}

template <int BITS, int TOK, bool OUT>
hipError_t launch_mx_stream(const ProjectArgs &a, const MxProduct &m, int n_cu, hipStream_t s) {
    const int n_rt = (a.n_a + a.n_b + kMxWeightTile - 1) / kMxWeightTile;
    const dim3 block(64 * kMxStreamWaves);
    // Two row tiles a workgroup where one would not fit the chip at once: 5120 ->
    // 14336 side by side, the whole call 11.6 us for one token and 13.8 for 32, by
    // one 13.4 and 16.9.
    if (n_rt > n_cu) hipLaunchKernelGGL((mx_stream_kernel<BITS, 2, TOK, OUT>), dim3((n_rt + 1) / 2), block, 0, s, a, m);
    else hipLaunchKernelGGL((mx_stream_kernel<BITS, 1, TOK, OUT>), dim3(n_rt), block, 0, s, a, m);
    return hipGetLastError();
}

// Up to 8 tokens leave the LDS to the weights: more of them on their way.  One
// token of 5120 -> 14336 side by side: the whole call 11.6 us, with room for 32
// tokens 11.9; the product of 8 and 9 tokens of 8 bits takes 9.1 and 10.5.
template <int BITS>
hipError_t launch_mx_stream(const ProjectArgs &a, const MxProduct &m, bool heads, int n_cu, hipStream_t s) {
    if (heads) return (a.n_tok <= 8 ? launch_mx_stream<BITS, 8, false> : launch_mx_stream<BITS, 32, false>)(a, m, n_cu, s);
    return (a.n_tok <= 8 ? launch_mx_stream<BITS, 8, true> : launch_mx_stream<BITS, 32, true>)(a, m, n_cu, s);
}

// The tiles, and what they take (us): to start and end, and for 256 values of
// k where a quarter of the CUs have a tile and where all do (the clock falls
// with the load), measured tile by tile.  Side by side, 2048 tokens of 5120 ->
// 14336 take 134 us by 256 x 256 and 152 by 128 x 256, of 4 bits 109 and 119;
// 6144 -> 5120 is 256 tiles of 128 x 320, but 320 of 128 x 256, 64 of them in a
// second round.
using MxLaunch = hipError_t (*)(const ProjectArgs &, const MxProduct &, hipStream_t);
struct MxForm {
    int bm, bn;
    float fixed, few, all;
    MxLaunch head, out, part;
};
template <int BITS, int BM, int BN, int WM, int WN, int S>
constexpr MxForm mx_form(float fixed, float few, float all) {
    using T = MxTile<BITS, BM, BN, WM, WN, S>;
    MxForm f{BM, BN, fixed, few, all, nullptr, launch_mx_gemm<T, kMxOut>, nullptr};
    if constexpr (BN == kHeadDim) f.head = launch_mx_gemm<T, kMxHead>;
    if constexpr (BM == 64 && BN == 128) f.part = launch_mx_gemm<T, kMxPart>;
    return f;
}
const MxForm kForms8[] = {
    mx_form<8, 256, 256, 2, 2, 3>(11.0f, 1.87f, 3.10f), mx_form<8, 128, 256, 2, 2, 4>(7.5f, 0.97f, 1.65f),
    mx_form<8, 64, 256, 2, 2, 4>(5.2f, 0.61f, 0.94f),   mx_form<8, 128, 320, 2, 2, 4>(8.0f, 1.17f, 2.20f),
    mx_form<8, 128, 128, 2, 2, 5>(5.5f, 0.65f, 0.95f),  mx_form<8, 64, 128, 1, 4, 6>(4.3f, 0.51f, 0.63f),
};
const MxForm kForms4[] = {
    mx_form<4, 256, 256, 2, 2, 2>(10.5f, 1.37f, 2.38f), mx_form<4, 128, 256, 2, 2, 3>(8.0f, 0.65f, 1.12f),
    mx_form<4, 64, 256, 2, 2, 3>(5.4f, 0.46f, 0.61f),   mx_form<4, 128, 320, 2, 2, 2>(8.0f, 1.01f, 1.63f),
    mx_form<4, 128, 128, 2, 2, 4>(4.9f, 0.42f, 0.69f),  mx_form<4, 64, 128, 1, 4, 6>(4.6f, 0.35f, 0.41f),
};
static_assert(std::size(kForms8) == std::size(kForms4), "one plan for both");

// n tiles of `nc` 256s on n_cu CUs: rounds of the chip, the last as full as it is.
double rounds_us(const MxForm &f, int64_t n, int nc, int n_cu) {
    const int64_t whole = n / n_cu;
    const double fill = static_cast<double>(n - whole * n_cu) / n_cu;
    double us = whole * (f.fixed + static_cast<double>(nc) * f.all);
    if (fill > 0) us += f.fixed + nc * (f.few + (f.all - f.few) * std::max(0.0, (fill - 0.25) / 0.75));
    return us;
}

}  // namespace

// Up to 32 tokens stream the weights past them; more take the tile, and split of
// hidden, of the least estimated time.  A split adds its partials, written and
// read back, and the finish launch.  At the border, 32 tokens streamed take 8.3
// us at 6144 -> 5120, 33 by four splits and their finish 7.6 + 3.1; with norm and
// RoPE at 5120 -> 14336 both need the finish, and take 12.2 and 11.4 before it.
bool plan_mx(const ProjectArgs &a, const MxProduct &m, bool heads, int n_cu, size_t part_floats, ProductPlan &plan) {
    const int T = a.n_tok, N = a.n_a + a.n_b;
    plan = ProductPlan{};
    plan.form = plan.pair = -1;
    plan.splits = 1;
    if (T <= kMxStreamTokens) {
        plan.stream = true;
        plan.partial = heads;
        return !heads || static_cast<size_t>(T) * N <= part_floats;
    }
    const MxForm *forms = m.bits == 8 ? kForms8 : kForms4;
    const int n512 = a.hidden / 512;
    double best_us = 0;
    for (int i = 0; i < static_cast<int>(std::size(kForms8)); ++i) {
        const MxForm &f = forms[i];
        if (heads && a.n_a % f.bn != 0) continue;  // a tile never straddles the two weights
        const int64_t tiles = static_cast<int64_t>((N + f.bn - 1) / f.bn) * ((T + f.bm - 1) / f.bm);
        for (int splits = 1; splits <= kGemmMaxSplits && splits <= n512; ++splits) {
            const bool partial = splits > 1 || (heads && !f.head);
            const double part = static_cast<double>(splits) * T * N;
            if (partial && (!f.part || part > static_cast<double>(part_floats))) break;
            double us = rounds_us(f, tiles * splits, 2 * ((n512 + splits - 1) / splits), n_cu);
            if (partial) us += 4.0 + 8.0 * part / 5.0e6;
            else if (heads) us += 0.02 * f.bm;  // norm, RoPE and three outputs' rows
            if (plan.form < 0 || us < best_us) {
                plan.form = i;
                plan.splits = splits;
                plan.partial = partial;
                best_us = us;
            }
        }
    }
    if (plan.form < 0) return false;
    plan.bm = forms[plan.form].bm;
    plan.bn = forms[plan.form].bn;
    return true;
}

hipError_t launch_mx_product(const ProjectArgs &args, const MxProduct &product, bool heads, int n_cu, const ProductPlan &plan,
                             hipStream_t s) {
    ProjectArgs a = args;
    MxProduct m = product;
    a.splits = plan.splits;
    hipError_t e = a.ev_before ? hipEventRecord(a.ev_before, s) : hipSuccess;
    if (e != hipSuccess) return e;
    if (plan.stream) {
        e = m.bits == 8 ? launch_mx_stream<8>(a, m, heads, n_cu, s) : launch_mx_stream<4>(a, m, heads, n_cu, s);
    } else {
        const MxForm &f = (m.bits == 8 ? kForms8 : kForms4)[plan.form];
        // Tiles that are normalised end some 6 us later than the others, of which
        // there are as many: where a CU takes a second tile, not two of them (5120
        // -> 14336 of 2048 tokens side by side: 127.5 us against 131, in 4 bits 107
        // against 111).  Tiles that all run at once keep the order of the heads
        // (181 tokens: 19.5 us against 19.7).
        m.by_kind = heads && static_cast<int64_t>((a.n_a + a.n_b) / f.bn) * ((a.n_tok + f.bm - 1) / f.bm) > n_cu;
        e = (plan.partial ? f.part : heads ? f.head : f.out)(a, m, s);
    }
    if (e != hipSuccess) return e;
    if (a.ev_after && (e = hipEventRecord(a.ev_after, s)) != hipSuccess) return e;
    if (!plan.partial) return hipSuccess;
    return heads ? launch_project_finish(a, true, s) : launch_out_finish(a, s);
}

}  // namespace kva
