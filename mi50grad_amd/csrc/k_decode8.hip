// GQA decode attention over the 8-bit cache (gfx950).
//
// out = softmax(q K^T / 16) V per query head over the values that the cache
// stands for (k_page8.h), as decode over the FP16 cache, with half its bytes.
// Stream-K over pages as there (k_walk.h): workgroup w walks the w-th share of
// the pages of all sequences, one wave per KV head; a sequence that the share
// holds whole is written out, a cut one leaves partials for the merge.
//
// A block is 8 KB in operand order, so a wave brings it in as eight 1 KB loads
// that write LDS directly (and one of its scales), through a ring of its own:
// no wave waits for another, and no register is held by a load in flight.
//   QK: S^T = K Q^T on 16x16x32 products, the codes as A (integers, exact),
//       the G query rows as columns of B; the block's scale goes into the
//       softmax's factor;
//   softmax: on the C layout (lane: head column l % 16, rows 4 (l / 16) .. + 3),
//       where four probabilities are already the B operand of
//   PV: O^T[dim][head] += V^T P^T on 16x16x16 products, V as values (code times
//       scale, exact in FP16).
// Both products run on the matrix unit: on the vector unit, as the FP16
// decode's PV, the conversion of the codes would come on top of six heads' sums.
#include "k_common.h"
#include "k_page8.h"
#include "k_walk.h"
#include "kva_internal.h"

namespace kva {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kQkScale = kLog2e / 16.0f;
// A column's reference max moves only when a block's passes it by more than
// this (log2 units): probabilities stay below 2^8, which FP16 holds to the same
// relative precision, and the accumulators are rescaled rarely.
constexpr float kSlack = 8.0f;
constexpr int kRing = 4;                              // blocks of LDS per wave
constexpr int kSlotBytes = 2 * kPageElems + 256;      // K, V, scales (one dword a lane)
constexpr int kLoads = 9;                             // vector loads of a block

__device__ __forceinline__ half8_t as_h8(uint4 v) { return __builtin_bit_cast(half8_t, v); }
__device__ __forceinline__ half4_t as_h4(uint2 v) { return __builtin_bit_cast(half4_t, v); }

// m: the reference max of this lane's head column, in log2 units; l: the
// FP16 probabilities of this lane's rows summed; acc: dims 16 t + 4 (l / 16) .. +
// 3 of the column's head.
struct State {
    float m, l;
    float4_t acc[16];
};
__device__ __forceinline__ void reset(State &st) {
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int t = 0; t < 16; ++t) st.acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
}

// Scores x (log2 units, masked ones -inf) of this lane's four rows to
// probabilities as the B operand.
__device__ __forceinline__ half4_t fold_scores(State &st, const float4_t &x) {
    constexpr uint32_t kOnes = 0x3c003c00u;  // FP16 pair (1, 1)
    const float mx = group4_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    const bool jump = mx > st.m + kSlack;
    if (__builtin_amdgcn_ballot_w64(jump)) {
        const float mn = jump ? mx : st.m;
        // From -inf, acc and l are zero; a column of NaN scores stays at -inf.
        const float corr = st.m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
        st.l *= corr;
#pragma unroll
        for (int t = 0; t < 16; ++t) st.acc[t] *= corr;
        st.m = mn;
    }
    const float mu = st.m == -INFINITY ? 0.0f : st.m;
    const uint32_t p0 = pack_p2(__builtin_amdgcn_exp2f(x[0] - mu), __builtin_amdgcn_exp2f(x[1] - mu));
    const uint32_t p1 = pack_p2(__builtin_amdgcn_exp2f(x[2] - mu), __builtin_amdgcn_exp2f(x[3] - mu));
    st.l = dot2(p1, kOnes, dot2(p0, kOnes, st.l));  // l sums the FP16 probabilities PV uses
    return as_h4(make_uint2(p0, p1));
}

// A full block from LDS.  Every read is requested before any is used.
__device__ __forceinline__ void fold_block(State &st, const uint8_t *slot, const uint4 (&qb)[8], int lane) {
    uint4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const uint4 *>(slot + 1024 * i + 16 * lane);
    const float2 sc = *reinterpret_cast<const float2 *>(slot + 2 * kPageElems);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4 *>(slot + kPageElems + 1024 * i + 16 * lane);
    __builtin_amdgcn_sched_barrier(0);
    float4_t s[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(codes8(k[i].x, k[i].y)), as_h8(qb[2 * i]), s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(codes8(k[i].z, k[i].w)), as_h8(qb[2 * i + 1]), s[1], 0, 0, 0);
    }
    const half4_t p = fold_scores(st, (s[0] + s[1]) * (sc.x * kQkScale));
    const uint32_t vs = scale_h2(sc.y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t ws[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int t = 0; t < 4; ++t)
            st.acc[4 * j + t] = __builtin_amdgcn_mfma_f32_16x16x16f16(as_h4(values4(ws[t], vs)), p, st.acc[4 * j + t], 0, 0, 0);
    }
}

// The open block: `lim` FP16 rows (1..15) in page order; what lies behind them
// is stale, so its scores are masked and its values zeroed.
__device__ __forceinline__ void fold_open(State &st, const uint16_t *open, const uint4 (&qb)[8], int lane, int lim) {
    const int grp = lane >> 4;
    float4_t s[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
    uint4 k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = ld16(open + 1024 * (i >> 1) + 16 * lane + 8 * (i & 1));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ld16(open + kPageElems + 1024 * (i >> 1) + 16 * lane + 8 * (i & 1));
#pragma unroll
    for (int i = 0; i < 8; ++i)
        s[i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(k[i]), as_h8(qb[i]), s[i & 1], 0, 0, 0);
    float4_t x = (s[0] + s[1]) * kQkScale;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 4 * grp + i < lim ? x[i] : -INFINITY;
    const half4_t p = fold_scores(st, x);
    const uint32_t m0 = (4 * grp < lim ? 0xffffu : 0u) | (4 * grp + 1 < lim ? 0xffff0000u : 0u);
    const uint32_t m1 = (4 * grp + 2 < lim ? 0xffffu : 0u) | (4 * grp + 3 < lim ? 0xffff0000u : 0u);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const uint4 w = v[t >> 1];  // dim tiles 2i, 2i + 1
        const uint2 y = (t & 1) ? make_uint2(w.z & m0, w.w & m1) : make_uint2(w.x & m0, w.y & m1);
        st.acc[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(as_h4(y), p, st.acc[t], 0, 0, 0);
    }
}

// B operand: query head col of the group (zero past G), k-step 2i + e holding
// dims 64 i + 16 (l / 16) + 8 e .. + 7.
__device__ __forceinline__ void load_query(uint4 (&qb)[8], const uint16_t *q, int G, int lane) {
    const int col = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        qb[k] = col < G ? ld16(q + col * kHeadDim + 64 * (k >> 1) + 16 * grp + 8 * (k & 1)) : make_uint4(0, 0, 0, 0);
}

// Eight loads of a block and one of its scales to a slot; off: the same
// loads through empty resources.
__device__ __forceinline__ void issue_block(uint32_t slot, const uint8_t *k, const uint8_t *v, const float *scales,
                                            bool on, int lane) {
    const auto rk = ro_rsrc(k, on ? kPageElems : 0u), rv = ro_rsrc(v, on ? kPageElems : 0u);
    const auto rs = ro_rsrc(scales, on ? 8u : 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_to_lds_at(rk, slot + 1024 * i, 16 * lane, 1024 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_to_lds_at(rv, slot + kPageElems + 1024 * i, 16 * lane, 1024 * i);
    touch_line(rs, slot + 2 * kPageElems, 4 * (lane & 1), 0);
}

// Held to 256 registers: with 512 the compiler keeps the accumulators in the
// other half and moves all 64 over at every block.
__global__ __launch_bounds__(64 * kDecodeHeadsPerWg, 2) void decode8_kernel(Decode8Args e) {
    const DecodeArgs &a = e.d;
    extern __shared__ __attribute__((aligned(16))) uint8_t ring[];  // [waves][kRing][kSlotBytes]
    const int w = blockIdx.x;
    int P, W;
    stream_k_shape(a, P, W);
    if (w >= W) return;
    const int p_begin = wg_start(w, P, W);
    const int p_end = wg_start(w + 1, P, W);
    if (p_begin >= p_end) return;
    const int hkv = a.num_kv_heads, nh = a.num_heads, G = nh / hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * (blockDim.x >> 6) + wave);
    const int lane = threadIdx.x & 63;
    const int col = lane & 15, grp = lane >> 4;
    uint8_t *mine = ring + static_cast<size_t>(wave) * kRing * kSlotBytes;

    // The first sequence of the share: the last with pages before it <= p_begin.
    int b0 = 0;
    for (int c0 = 0; c0 < a.n_seqs; c0 += 64) {
        const int i = c0 + lane;
        const uint64_t before = __ballot((i < a.n_seqs ? a.pre_seq[i + 1] : INT32_MAX) <= p_begin);
        b0 += __popcll(before);
        if (before != ~0ull) break;
    }
    b0 = __builtin_amdgcn_readfirstlane(b0);
    // A sequence's pages in the share: [p0, p1) of its npg, the full ones before
    // `full`; only its last page can be open.  (Every field is wave-uniform.)
    struct Segment {
        int b, p0, p1, npg, ctx, full;
        const int32_t *row;
    };
    auto segment = [&](int b) -> Segment {
        Segment g;
        g.b = b;
        g.ctx = ld_uniform(a.ctx_lens + b);
        const int base = ld_uniform(a.pre_seq + b);
        g.row = a.table + static_cast<size_t>(ld_uniform(a.seq_ids + b)) * a.table_stride;
        g.npg = (g.ctx + kBlockTokens - 1) / kBlockTokens;
        g.p0 = max(0, p_begin - base);
        g.p1 = min(g.npg, p_end - base);
        g.full = min(g.p1, g.ctx / kBlockTokens);
        return g;
    };
    // The issue side, kRing - 1 full pages ahead of the products across
    // sequences: page ip of segment ig next, whose id is `id`; past the share the
    // same loads go through empty resources, so the load counter advances alike.
    const int b_last = [&] {  // the sequence of the share's last page
        int b = b0;
        while (ld_uniform(a.pre_seq + b + 1) < p_end) ++b;
        return b;
    }();
    Segment ig = segment(b0);
    int ip = ig.p0, id = 0;
    bool on = true;
    auto settle = [&]() {  // to the next full page of the share, if there is one
        while (ip >= ig.full) {
            if (ig.b >= b_last) {
                on = false;
                return;
            }
            ig = segment(ig.b + 1);
            ip = ig.p0;
        }
    };
    auto fetch = [&]() {
        if (on) id = ld_uniform(ig.row + ip);
    };
    auto issue = [&](int slot) {
        const size_t blk = static_cast<size_t>(id) * hkv + h;
        issue_block(__builtin_amdgcn_readfirstlane(lds_addr(mine + slot * kSlotBytes)), e.k8 + blk * kPageElems, e.v8 + blk * kPageElems,
                    e.scales + 2 * blk, on, lane);
        if (on) {
            ++ip;
            settle();
        }
    };
    settle();
#pragma unroll
    for (int i = 0; i + 1 < kRing; ++i) {
        fetch();
        issue(i);
    }
    fetch();

    int n = 0;  // blocks folded in: the next is in slot n % kRing
    for (int b = b0; b <= b_last; ++b) {
        const Segment g = segment(b);
        if (g.p0 >= g.p1) continue;
        uint4 qb[8];
        load_query(qb, a.q + (static_cast<size_t>(b) * nh + h * G) * kHeadDim, G, lane);
        // Taken in here: left to the compiler, the wait would sit in front of every
        // block's products and, not seeing the loads to LDS, drain the ring there.
#pragma unroll
        for (int k = 0; k < 8; ++k) asm volatile("" : "+v"(qb[k].x), "+v"(qb[k].y), "+v"(qb[k].z), "+v"(qb[k].w));
        State st;
        reset(st);
#pragma unroll 1
        for (int p = g.p0; p < g.full; ++p, ++n) {
            // The last reads of the slot that is issued over have returned, and
            // the page id is there.
            __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0)
            __builtin_amdgcn_sched_barrier(0);
            issue((n + kRing - 1) % kRing);
            wait_vm<kLoads * (kRing - 1)>();
            __builtin_amdgcn_sched_barrier(0);
            fold_block(st, mine + (n % kRing) * kSlotBytes, qb, lane);
            // Behind the block's LDS reads: a scalar load in flight makes each of
            // their waits a wait for all.
            __builtin_amdgcn_sched_barrier(0);
            fetch();
        }
        if (g.full < g.p1)
            fold_open(st, e.open + (static_cast<size_t>(ld_uniform(e.open_slot + b)) * hkv + h) * 2 * kPageElems, qb, lane,
                      g.ctx & 15);
        const float lt = group4_sum(st.l);  // the four lane groups hold disjoint rows
        if (g.p0 == 0 && g.p1 == g.npg && col < G) {
            const float inv = 1.0f / lt;
            uint16_t *o = a.out + (static_cast<size_t>(b) * nh + h * G + col) * kHeadDim + 4 * grp;
            const uint16_t *gate =
                a.gate ? a.gate + static_cast<int64_t>(b) * a.gate_stride + (h * G + col) * kHeadDim + 4 * grp : nullptr;
            uint2 gw[16];
            if (gate) {
#pragma unroll
                for (int t = 0; t < 16; ++t) gw[t] = ld8(gate + 16 * t);
            }
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const float4_t y = st.acc[t] * inv;
                *reinterpret_cast<uint2 *>(o + 16 * t) =
                    gate ? gate4(y[0], y[1], y[2], y[3], gw[t]) : pack_out4(y[0], y[1], y[2], y[3]);
            }
        } else if (col < G) {
            const int slot = 2 * w + (b == b0 ? 0 : 1);
            const size_t u = (static_cast<size_t>(slot) * hkv + h) * G + col;
#pragma unroll
            for (int t = 0; t < 16; ++t)
                *reinterpret_cast<float4_t *>(a.ws_acc + u * kHeadDim + 16 * t + 4 * grp) = st.acc[t];
            if (grp == 0) {
                a.ws_ml[u * 2] = st.m;
                a.ws_ml[u * 2 + 1] = lt;
            }
        }
    }
    // Loads past the share write LDS too: none may land after it is handed on.
    __builtin_amdgcn_s_waitcnt(0);
}

}  // namespace

hipError_t launch_decode8(const Decode8Args &a, hipStream_t s) {
    const DecodeArgs &d = a.d;
    if (d.n_seqs <= 0) return hipSuccess;
    int hpw = d.num_kv_heads <= kDecodeHeadsPerWg ? d.num_kv_heads : kDecodeHeadsPerWg;
    while (d.num_kv_heads % hpw) --hpw;
    const size_t lds = static_cast<size_t>(hpw) * kRing * kSlotBytes;
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(decode8_kernel),
                                       hipFuncAttributeMaxDynamicSharedMemorySize,
                                       kDecodeHeadsPerWg * kRing * kSlotBytes);
    if (e != hipSuccess) return e;
    if (d.ev_before && (e = hipEventRecord(d.ev_before, s)) != hipSuccess) return e;
    hipLaunchKernelGGL(decode8_kernel, dim3(d.n_wg, d.num_kv_heads / hpw), dim3(64 * hpw), lds, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (d.ev_after && (e = hipEventRecord(d.ev_after, s)) != hipSuccess) return e;
    return launch_decode_merge(d, s);
}

}  // namespace kva
