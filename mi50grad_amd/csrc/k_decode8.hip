// GQA decode attention over the 8-bit cache (gfx950).
//
// out = softmax(q K^T / 16) V per query head over the values that the cache
// stands for (k_page8.h), as decode over the FP16 cache, with half its bytes.
// Stream-K over pages as there (k_walk.h): workgroup w walks the w-th share of
// the pages of all sequences, one wave per KV head; a sequence that the share
// holds whole is written out, a cut one leaves partials for the merge.  Short
// steps take a workgroup per sequence and KV head instead (whole8_kernel).
//
// What bounds it is HBM: 48 sequences of 4096 to 32768 rows (20800 in the mean,
// 2.05 GB) take 355 us, 5.8 TB/s; 32 of 1024 to 8192 (4300 in the mean, 285 MB)
// 63 us, some 14 us of it the start (three waits for memory in turn), the tail
// and the merge.  That is with four KV heads; a workgroup has a wave per KV head,
// four at most, and its ring leaves room for one of four waves to a CU.  The 32
// sequences with eight KV heads (two rounds of workgroups) take 115 us where their
// bytes take 96, with two 44 (24), with one, a wave to a CU, 39 (12).
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
// probabilities as the B operand.  They are rounded to FP16, which the products
// take: with sums in FP32 over the rounded ones an output is off by 2.9e-4
// (root mean square, relative), 2.1e-4 of it its own rounding to FP16.
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

// The step's sequences as the walk reads them.
struct StepRefs {
    const int32_t *pre_seq, *ctx_lens, *seq_ids, *open_slot, *table;
    int32_t table_stride, n_seqs;
};

// A sequence's pages in a share: [p0, p1) of its npg, those before `full` not
// open.
struct Segment {
    int b, p0, p1, npg, ctx, full, base, slot;
    const int32_t *row;
};

// A share [p_begin, p_end) of the step's pages, its sequences b0 .. b_last.  What
// is known of 64 sequences lies in the lanes of four registers, loaded
// together, so a walk of few sequences waits for memory once for all of it.
struct Share {
    StepRefs r;
    int p_begin, p_end, b0, b_last;
    int win;                   // the lanes' first sequence
    int ctx, pre, sid, slot;   // lane l: of sequence win + l

    __device__ __forceinline__ void window(int b, int lane) {
        win = b;
        const int i = min(b + lane, r.n_seqs - 1);
        ctx = r.ctx_lens[i];
        pre = r.pre_seq[i];
        sid = r.seq_ids[i];
        slot = r.open_slot[i];
        // Taken in here, so that no later use waits for loads in flight.
        asm volatile("" : "+v"(ctx), "+v"(pre), "+v"(sid), "+v"(slot));
    }
    // False: the share is empty.
    __device__ __forceinline__ bool begin(const StepRefs &refs, int w, int P, int W, int lane) {
        r = refs;
        p_begin = wg_start(w, P, W);
        p_end = wg_start(w + 1, P, W);
        if (p_begin >= p_end) return false;
        // The last sequence that begins at or before the share, and the last
        // before its end: 64 at a time (empty ones share their beginning with the next).
        b0 = 0;
        for (int g = 0; g < r.n_seqs; g += 64) {
            window(g, lane);
            const uint64_t there = r.n_seqs - g >= 64 ? ~0ull : (1ull << (r.n_seqs - g)) - 1;
            const int n = __popcll(__ballot(pre <= p_begin) & there);
            if (n > 0) b0 = g + n - 1;
            if (n < 64) break;
        }
        if (b0 < win) window(b0, lane);
        b_last = b0 = __builtin_amdgcn_readfirstlane(b0);
        const uint64_t there = r.n_seqs - win >= 64 ? ~0ull : (1ull << (r.n_seqs - win)) - 1;
        b_last = __builtin_amdgcn_readfirstlane(win + __popcll(__ballot(pre < p_end) & there) - 1);
        while (b_last + 1 < r.n_seqs && b_last == win + 63 && ld_uniform(r.pre_seq + b_last + 1) < p_end) {
            window(b_last + 1, lane);
            const uint64_t more = r.n_seqs - win >= 64 ? ~0ull : (1ull << (r.n_seqs - win)) - 1;
            b_last = __builtin_amdgcn_readfirstlane(win + __popcll(__ballot(pre < p_end) & more) - 1);
        }
        if (b0 < win) window(b0, lane);
        return true;
    }
    __device__ __forceinline__ Segment at(int b) const {
        Segment g;
        g.b = b;
        int s;
        if (b - win < 64) {
            g.ctx = __builtin_amdgcn_readlane(ctx, b - win);
            g.base = __builtin_amdgcn_readlane(pre, b - win);
            g.slot = __builtin_amdgcn_readlane(slot, b - win);
            s = __builtin_amdgcn_readlane(sid, b - win);
        } else {
            g.ctx = ld_uniform(r.ctx_lens + b);
            g.base = ld_uniform(r.pre_seq + b);
            g.slot = ld_uniform(r.open_slot + b);
            s = ld_uniform(r.seq_ids + b);
        }
        g.row = r.table + static_cast<size_t>(s) * r.table_stride;
        g.npg = (g.ctx + kBlockTokens - 1) / kBlockTokens;
        g.p0 = max(0, p_begin - g.base);
        g.p1 = min(g.npg, p_end - g.base);
        g.full = min(g.p1, g.ctx / kBlockTokens);
        return g;
    }
};

// The issue side of the walk: the share's full pages in order, across
// sequences.  `id` is the next one's, fetched a page ahead by a scalar load,
// the first 64 by one vector load together.
struct PageFeed {
    Segment g;
    int ip, id, first, n_first;  // n_first pages from `first` of the first sequence are in ids
    int ids;
    bool on;

    __device__ __forceinline__ void settle(const Share &sh) {  // to the next page, if there is one
        while (ip >= g.full) {
            if (g.b >= sh.b_last) {
                on = false;
                return;
            }
            g = sh.at(g.b + 1);
            ip = g.p0;
            n_first = 0;
        }
    }
    // Requests the first ids; take() before fetch().
    __device__ __forceinline__ void begin(const Share &sh, int lane) {
        g = sh.at(sh.b0);
        ip = g.p0;
        on = true;
        id = 0;
        n_first = 64;
        settle(sh);
        n_first = on ? 64 : 0;
        first = ip;
        ids = on ? g.row[min(ip + lane, g.npg - 1)] : 0;
    }
    __device__ __forceinline__ void take() { asm volatile("" : "+v"(ids)); }
    __device__ __forceinline__ void fetch() {
        if (!on) return;
        if (n_first && ip - first < n_first)
            id = __builtin_amdgcn_readlane(ids, ip - first);
        else
            id = ld_uniform(g.row + ip);
    }
    __device__ __forceinline__ void next(const Share &sh) {
        if (!on) return;
        ++ip;
        settle(sh);
    }
};

// Held to 256 registers: with 512 the compiler keeps the accumulators in the
// other half and moves all 64 over at every block.
__global__ __launch_bounds__(64 * kDecodeHeadsPerWg, 2) void decode8_kernel(Decode8Args e) {
    const DecodeArgs &a = e.d;
    extern __shared__ __attribute__((aligned(16))) uint8_t ring[];  // [waves][kRing][kSlotBytes]
    const int w = blockIdx.x;
    int P, W;
    stream_k_shape(a, P, W);
    if (w >= W) return;
    const int hkv = a.num_kv_heads, nh = a.num_heads, G = nh / hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * (blockDim.x >> 6) + wave);
    const int lane = threadIdx.x & 63;
    const int col = lane & 15, grp = lane >> 4;
    uint8_t *mine = ring + static_cast<size_t>(wave) * kRing * kSlotBytes;

    // A workgroup starts with three waits for memory: the sequences' facts, the
    // first page ids with the first query rows, the first blocks.
    Share share;
    if (!share.begin({a.pre_seq, a.ctx_lens, a.seq_ids, e.open_slot, a.table, a.table_stride, a.n_seqs}, w, P, W, lane)) return;
    const int b0 = share.b0;
    uint4 qb[8];
    auto query = [&](int b) { load_query(qb, a.q + (static_cast<size_t>(b) * nh + h * G) * kHeadDim, G, lane); };
    // Taken in before the blocks' loads go out (a sequence's first wait): left to
    // the compiler, the wait would sit in front of every block's products and, not
    // seeing the loads to LDS, drain the ring there.
    auto take_query = [&]() {
#pragma unroll
        for (int k = 0; k < 8; ++k) asm volatile("" : "+v"(qb[k].x), "+v"(qb[k].y), "+v"(qb[k].z), "+v"(qb[k].w));
    };
    // kRing - 1 blocks ahead of the products; past the share the same loads go
    // through empty resources, so the load counter advances alike.
    PageFeed feed;
    feed.begin(share, lane);
    query(b0);
    feed.take();
    take_query();
    auto issue = [&](int slot) {
        const size_t blk = static_cast<size_t>(feed.id) * hkv + h;
        issue_block(__builtin_amdgcn_readfirstlane(lds_addr(mine + slot * kSlotBytes)), e.k8 + blk * kPageElems,
                    e.v8 + blk * kPageElems, e.scales + 2 * blk, feed.on, lane);
        feed.next(share);
    };
#pragma unroll
    for (int i = 0; i + 1 < kRing; ++i) {
        feed.fetch();
        issue(i);
    }
    feed.fetch();

    int n = 0;  // blocks folded in: the next is in slot n % kRing
    for (int b = b0; b <= share.b_last; ++b) {
        const Segment g = share.at(b);
        if (g.p0 >= g.p1) continue;
        if (b > b0) {
            query(b);
            take_query();
        }
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
            feed.fetch();
        }
        if (g.full < g.p1)
            fold_open(st, e.open + (static_cast<size_t>(g.slot) * hkv + h) * 2 * kPageElems, qb, lane,
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

// ---- short steps: a workgroup per sequence and KV head ----
//
// Its waves take the sequence's pages in turn and merge in LDS: no partials, no
// second launch, and at the start one wait for memory fewer (the step plan holds
// the ids of the first pages).  The wave that has the fewest pages takes the open
// block, before its others, while those are on their way.
constexpr int kShortWaves = 8, kShortRing = 2;
constexpr int kShortLds = kShortWaves * kShortRing * kSlotBytes;
static_assert(kShortWaves * 8 * kHeadDim * 4 <= kShortLds, "eight heads' accumulators of every wave take the ring's place");

__global__ __launch_bounds__(64 * kShortWaves) void whole8_kernel(Decode8Args e) {
    extern __shared__ __attribute__((aligned(16))) uint8_t ring[];  // [waves][kShortRing][kSlotBytes]
    __shared__ float2 ml[kShortWaves][16];
    const DecodeArgs &a = e.d;
    const int hkv = a.num_kv_heads, nh = a.num_heads, G = nh / hkv;
    const int b = blockIdx.x / hkv, h = blockIdx.x - b * hkv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    uint8_t *mine = ring + static_cast<size_t>(wave) * kShortRing * kSlotBytes;

    // The wave's i-th page is wave + kShortWaves i; lane l: the id of page i0 + l of
    // its own, the first ones from the plan.
    constexpr int kPlanned = kPlanPages / kShortWaves;
    int ids = lane < kPlanned ? a.plan_pages[b * kPlanPages + wave + kShortWaves * lane] : 0, i0 = 0;
    uint4 qb[8];
    load_query(qb, a.q + (static_cast<size_t>(b) * nh + h * G) * kHeadDim, G, lane);
    const int ctx = ld_uniform(a.ctx_lens + b), slot_open = ld_uniform(e.open_slot + b);
    const int32_t *row = a.table + static_cast<size_t>(ld_uniform(a.seq_ids + b)) * a.table_stride;
    asm volatile("" : "+v"(ids));
#pragma unroll
    for (int k = 0; k < 8; ++k) asm volatile("" : "+v"(qb[k].x), "+v"(qb[k].y), "+v"(qb[k].z), "+v"(qb[k].w));
    const int full = ctx / kBlockTokens;  // pages that are not open
    const int n = full > wave ? (full - wave + kShortWaves - 1) / kShortWaves : 0;  // this wave's
    auto table_ids = [&](int from, int skip) {
        if (lane >= skip) ids = row[min(wave + kShortWaves * (from + lane), full - 1)];
        asm volatile("" : "+v"(ids));
    };
    if (n > kPlanned) table_ids(0, kPlanned);
    auto issue = [&](int i) {
        if (i - i0 == 64 && i < n) {
            i0 = i;
            table_ids(i, 0);
        }
        const size_t blk = static_cast<size_t>(__builtin_amdgcn_readlane(ids, min(i - i0, 63))) * hkv + h;
        issue_block(__builtin_amdgcn_readfirstlane(lds_addr(mine + i % kShortRing * kSlotBytes)), e.k8 + blk * kPageElems,
                    e.v8 + blk * kPageElems, e.scales + 2 * blk, i < n, lane);
    };
#pragma unroll
    for (int i = 0; i + 1 < kShortRing; ++i) issue(i);
    State st;
    reset(st);
    if ((ctx & 15) && wave == full % kShortWaves)
        fold_open(st, e.open + (static_cast<size_t>(slot_open) * hkv + h) * 2 * kPageElems, qb, lane, ctx & 15);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0): the slot's last reads have returned
        __builtin_amdgcn_sched_barrier(0);
        issue(i + kShortRing - 1);
        wait_vm<kLoads * (kShortRing - 1)>();
        __builtin_amdgcn_sched_barrier(0);
        fold_block(st, mine + i % kShortRing * kSlotBytes, qb, lane);
    }
    const float lt = group4_sum(st.l);
    // No load may land in the ring any more, nor may a wave still read it.
    wait_vm_lds<0>();
    __syncthreads();
    float *acc = reinterpret_cast<float *>(ring);  // [wave][G][256]
    if (col < G) {
        float *to = acc + (wave * G + col) * kHeadDim + 4 * grp;
#pragma unroll
        for (int t = 0; t < 16; ++t) *reinterpret_cast<float4_t *>(to + 16 * t) = st.acc[t];
        if (grp == 0) ml[wave][col] = make_float2(st.m, lt);
    }
    __syncthreads();
    // Four dims to a thread.
    for (int i = threadIdx.x; i < G * (kHeadDim / 4); i += 64 * kShortWaves) {
        const int g = i / (kHeadDim / 4), d = 4 * (i % (kHeadDim / 4)), hq = h * G + g;
        const uint2 gw =
            a.gate ? ld8(a.gate + static_cast<int64_t>(b) * a.gate_stride + hq * kHeadDim + d) : make_uint2(0, 0);
        float big = -INFINITY;
#pragma unroll
        for (int w = 0; w < kShortWaves; ++w) big = fmaxf(big, ml[w][g].x);
        // A head whose every score is NaN stays at -inf, its sum NaN.
        const float mu = big == -INFINITY ? 0.0f : big;
        float l = 0.0f;
        float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kShortWaves; ++w) {
            const float2 x = ml[w][g];
            // At -inf: a wave without pages (zeros), or NaN sums that stay.
            const float c = x.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x.x - mu);
            l += c * x.y;
            o += c * *reinterpret_cast<const float4_t *>(acc + (w * G + g) * kHeadDim + d);
        }
        o *= 1.0f / l;
        *reinterpret_cast<uint2 *>(a.out + (static_cast<size_t>(b) * nh + hq) * kHeadDim + d) =
            a.gate ? gate4(o[0], o[1], o[2], o[3], gw) : pack_out4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace

hipError_t launch_decode8(const Decode8Args &a, hipStream_t s) {
    const DecodeArgs &d = a.d;
    if (d.n_seqs <= 0) return hipSuccess;
    if (d.whole) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(whole8_kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kShortLds);
        if (e != hipSuccess) return e;
        if (d.ev_before && (e = hipEventRecord(d.ev_before, s)) != hipSuccess) return e;
        hipLaunchKernelGGL(whole8_kernel, dim3(d.n_seqs * d.num_kv_heads), dim3(64 * kShortWaves), kShortLds, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        return d.ev_after ? hipEventRecord(d.ev_after, s) : hipSuccess;
    }
    const int hpw = heads_per_wg(d.num_kv_heads);
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
