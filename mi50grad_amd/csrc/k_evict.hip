// Eviction by accumulated attention weight, over FP16 and 8-bit caches (gfx950):
// what the step's last tokens look at (stats_kernel, sum_kernel), which rows
// stay (select_kernel), and those rows in pages of their own (gather_kernel).
//
// Weights.  For a sequence's last m = min(new tokens, n_obs) tokens and the G
// query heads of a KV head: w[row] = decay * w[row] + sum over (token, head) of
// softmax(q K^T / 16)[row], each token seeing rows up to its own.  Two passes
// over K: the first leaves every query row's max and sum, the second the
// probabilities, summed.  Query rows are (token, head) pairs, 16 to a tile, the
// operand B of 16x16x32 products, in LDS for the whole workgroup; a wave takes a
// page as A and multiplies it with every tile.  In the C layout a lane holds
// one query row (column l % 16) and four keys (4 (l / 16) .. + 3), so the max and
// sum of the first pass stay in the lane until the end, and the second pass
// sums its tiles in the lane before the sixteen lanes of a row once per page.
#include "k_common.h"
#include "k_page8.h"
#include "kva_internal.h"

namespace kva {
namespace {

constexpr float kQkScale = 1.4426950408889634f / 16.0f;
constexpr int kWeightWaves = 4;

__device__ __forceinline__ half8_t as_h8(uint4 v) { return __builtin_bit_cast(half8_t, v); }

// Sum over the 16 lanes of a DPP row; every lane gets the sum.
__device__ __forceinline__ float row16_sum(float x) {
    x += dpp_f<kDppQuadXor1>(x);
    x += dpp_f<kDppQuadXor2>(x);
    x += dpp_f<kDppRowHalfMirror>(x);
    x += dpp_f<kDppRowMirror>(x);
    return x;
}

// A page's keys as this lane's part of A: row l % 16, and the dims that the
// lane's B holds at each k-step (FP16: 64 (l / 16) + 8 s .. + 7; 8-bit cache:
// 64 (s / 2) + 16 (l / 16) + 8 (s % 2) .. + 7).  raw: what memory holds of them.
template <bool kInt8>
struct Keys {
    uint4 raw[kInt8 ? 4 : 8];
    float factor;  // of the scores, log2(e) / 16 included
};
template <bool kInt8>
__device__ __forceinline__ int query_dim(int s, int grp) {
    return kInt8 ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 64 * grp + 8 * s;
}

// What a workgroup works on: pages [p0, p1) of sequence b for KV head h.
struct Span {
    int b, h, sid, slot, ctx, obs, tok, p0, p1;  // slot: open block; obs: query tokens, from token `tok` of the step
};
__device__ __forceinline__ Span span_of(const WeightArgs &a) {
    Span s;
    s.b = blockIdx.z;
    s.h = blockIdx.y;
    s.sid = ld_uniform(a.seq_ids + s.b);
    s.slot = a.k8 ? ld_uniform(a.open_slot + s.b) : 0;
    s.ctx = ld_uniform(a.ctx_lens + s.b);
    const int t0 = ld_uniform(a.tok_off + s.b), t1 = ld_uniform(a.tok_off + s.b + 1);
    s.obs = min(t1 - t0, a.n_obs);
    s.tok = t1 - s.obs;
    const int n = (s.ctx + kBlockTokens - 1) / kBlockTokens;
    s.p0 = floor_muldiv(blockIdx.x, n, gridDim.x);
    s.p1 = floor_muldiv(blockIdx.x + 1, n, gridDim.x);
    return s;
}

template <bool kInt8>
__device__ __forceinline__ void load_keys(Keys<kInt8> &k, const WeightArgs &a, const Span &s, int page, int id, int lane) {
    const int hkv = a.num_kv_heads;
    if constexpr (kInt8) {
        const size_t b = static_cast<size_t>(id) * hkv + s.h;
        const uint8_t *src = a.k8 + b * kPageElems + 16 * lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) k.raw[i] = *reinterpret_cast<const uint4 *>(src + 1024 * i);
        k.factor = a.scales[2 * b] * kQkScale;
    } else {
        const uint16_t *src =
            a.k_pool + ((static_cast<size_t>(id) * kBlockTokens + (lane & 15)) * hkv + s.h) * kHeadDim + 64 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) k.raw[i] = ld16(src + 8 * i);
        k.factor = kQkScale;
    }
}
template <bool kInt8>
__device__ __forceinline__ void operands(half8_t (&op)[8], float &factor, const Keys<kInt8> &k, const WeightArgs &a,
                                         const Span &s, int page, int lane) {
    factor = k.factor;
    if constexpr (kInt8) {
        if (page == (s.ctx >> 4)) {  // the open page
            const uint16_t *src = a.open + (static_cast<size_t>(s.slot) * a.num_kv_heads + s.h) * 2 * kPageElems + 16 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) op[i] = as_h8(ld16(src + 1024 * (i >> 1) + 8 * (i & 1)));
            factor = kQkScale;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                op[2 * i] = as_h8(codes8(k.raw[i].x, k.raw[i].y));
                op[2 * i + 1] = as_h8(codes8(k.raw[i].z, k.raw[i].w));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) op[i] = as_h8(k.raw[i]);
    }
}

// The span's query rows to LDS as B operands: [tile][k-step][lane] of 16 bytes,
// zeros past the last row.
template <bool kInt8>
__device__ __forceinline__ void load_queries(uint4 *qs, const WeightArgs &a, const Span &s, int tiles) {
    const int G = a.num_heads / a.num_kv_heads;
    for (int i = threadIdx.x; i < tiles * 512; i += blockDim.x) {
        const int lane = i & 63, step = (i >> 6) & 7, row = 16 * (i >> 9) + (lane & 15);
        const int iq = row / G;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (iq < s.obs)
            x = ld16(a.q + (static_cast<size_t>(s.tok + iq) * a.num_heads + s.h * G + row - iq * G) * kHeadDim +
                     query_dim<kInt8>(step, lane >> 4));
        qs[i] = x;
    }
}

// Walks the span's pages, this wave's in turn: scores(t, x) gets tile t's in
// log2 units, -inf where the row does not see the key; done(page) ends a page.
template <bool kInt8, int NT, class Scores, class Done>
__device__ __forceinline__ void walk(const WeightArgs &a, const Span &s, const uint4 *qs, int tiles, Scores scores,
                                     Done done) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.num_heads / a.num_kv_heads;
    const int32_t *row = a.table + static_cast<size_t>(s.sid) * a.table_stride;
    const int last = s.p1 - 1;
    int p = s.p0 + wave;
    if (p > last) return;
    // The last key that this lane's query row of each tile sees.
    int see[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int iq = (16 * t + col) / G;
        see[t] = iq < s.obs ? s.ctx - s.obs + iq : -1;
    }
    Keys<kInt8> cur, nxt;
    load_keys(cur, a, s, p, ld_uniform(row + p), lane);
    int id = ld_uniform(row + min(p + kWeightWaves, last));
    for (; p <= last; p += kWeightWaves) {
        load_keys(nxt, a, s, min(p + kWeightWaves, last), id, lane);
        id = ld_uniform(row + min(p + 2 * kWeightWaves, last));
        half8_t op[8];
        float factor;
        operands<kInt8>(op, factor, cur, a, s, p, lane);
        const bool whole = 16 * p + 15 <= s.ctx - s.obs;  // every query row sees every key
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t >= tiles) continue;  // uniform
            float4_t x = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                x = __builtin_amdgcn_mfma_f32_16x16x32_f16(op[k], as_h8(qs[(t * 8 + k) * 64 + lane]), x, 0, 0, 0);
            x *= factor;
            if (!whole || 16 * t + 15 >= s.obs * G) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = 16 * p + 4 * grp + i <= see[t] ? x[i] : -INFINITY;
            }
            scores(t, x);
        }
        done(p);
        cur = nxt;
    }
}

// (m, l) of every query row over the span's pages: part[b][h][split][row].
template <bool kInt8, int NT>
__global__ __launch_bounds__(64 * kWeightWaves) void stats_kernel(WeightArgs a) {
    __shared__ uint4 qs[NT * 512];
    __shared__ float2 wave_ml[kWeightWaves][NT * 16];
    const Span s = span_of(a);
    if (s.obs == 0) return;
    const int rows = s.obs * (a.num_heads / a.num_kv_heads), tiles = (rows + 15) / 16;
    load_queries<kInt8>(qs, a, s, tiles);
    __syncthreads();
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
    }
    walk<kInt8, NT>(
        a, s, qs, tiles,
        [&](int t, const float4_t &x) {
            const float mn = fmaxf(m[t], fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            const float mu = mn == -INFINITY ? 0.0f : mn;
            l[t] = l[t] * __builtin_amdgcn_exp2f(m[t] - mu) + (__builtin_amdgcn_exp2f(x[0] - mu) + __builtin_amdgcn_exp2f(x[1] - mu)) +
                   (__builtin_amdgcn_exp2f(x[2] - mu) + __builtin_amdgcn_exp2f(x[3] - mu));
            m[t] = mn;
        },
        [](int) {});
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t >= tiles) continue;
        const float mx = group4_max(m[t]);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float lt = group4_sum(l[t] * __builtin_amdgcn_exp2f(m[t] - mu));
        if (lane < 16) wave_ml[wave][16 * t + lane] = make_float2(mx, lt);
    }
    __syncthreads();
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
        float mx = -INFINITY, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < kWeightWaves; ++w) mx = fmaxf(mx, wave_ml[w][r].x);
        const float mu = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < kWeightWaves; ++w) lt += wave_ml[w][r].y * __builtin_amdgcn_exp2f(wave_ml[w][r].x - mu);
        a.part[((static_cast<size_t>(s.b) * a.num_kv_heads + s.h) * gridDim.x + blockIdx.x) * a.part_rows + r] =
            make_float2(mx, lt);
    }
}

// The probabilities of the span's rows, summed over the query rows, onto the
// decayed weights.
template <bool kInt8, int NT>
__global__ __launch_bounds__(64 * kWeightWaves) void sum_kernel(WeightArgs a) {
    __shared__ uint4 qs[NT * 512];
    __shared__ float2 stat[NT * 16];
    const Span s = span_of(a);
    const int rows = s.obs * (a.num_heads / a.num_kv_heads), tiles = (rows + 15) / 16;
    load_queries<kInt8>(qs, a, s, tiles);
    for (int r = threadIdx.x; r < NT * 16; r += blockDim.x) {
        float mx = -INFINITY, lt = 0.0f;
        if (r < rows) {
            const float2 *part = a.part + (static_cast<size_t>(s.b) * a.num_kv_heads + s.h) * gridDim.x * a.part_rows + r;
            for (int i = 0; i < static_cast<int>(gridDim.x); ++i) mx = fmaxf(mx, part[static_cast<size_t>(i) * a.part_rows].x);
            const float mu = mx == -INFINITY ? 0.0f : mx;
            for (int i = 0; i < static_cast<int>(gridDim.x); ++i) {
                const float2 p = part[static_cast<size_t>(i) * a.part_rows];
                lt += p.y * __builtin_amdgcn_exp2f(p.x - mu);
            }
        }
        stat[r] = make_float2(mx, 1.0f / lt);
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    float m[NT], inv[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float2 x = stat[16 * t + col];
        m[t] = x.x == -INFINITY ? 0.0f : x.x;
        inv[t] = x.y;
    }
    float *w = a.weights + (static_cast<size_t>(s.b) * a.num_kv_heads + s.h) * a.w_stride;
    float4_t sum = float4_t{0.f, 0.f, 0.f, 0.f};
    walk<kInt8, NT>(
        a, s, qs, tiles,
        [&](int t, const float4_t &x) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[i] += x[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[i] - m[t]) * inv[t];
        },
        [&](int page) {
            float mine = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float all = row16_sum(sum[i]);
                mine = col == i ? all : mine;
            }
            sum = float4_t{0.f, 0.f, 0.f, 0.f};
            const int key = 16 * page + 4 * grp + col;
            if (col < 4 && key < s.ctx) w[key] = a.decay == 0.0f ? mine : fmaf(a.decay, w[key], mine);
        });
}

// ---- which rows stay ---------------------------------------------------------

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// Larger weights have larger keys; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w == w ? w + 0.0f : -INFINITY);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A workgroup per (sequence and KV head, layer).  The key of the last row that
// stays is found by its digits (12, 10 and 10 bits, the first with sign, exponent
// and three bits of the significand, so that weights of a few binades spread
// over many counters); then the rows above it, and as many of its equals from
// the lowest place on as there is room for, are written in order.  kLds: the
// keys are held in LDS (up to kSelectLds rows), else read again for each step.
template <bool kLds>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[4096];
    __shared__ int wave_sum[kSelectWaves + 1], wave_tie[kSelectWaves + 1];
    __shared__ int found[2];
    const int u = blockIdx.x, layer = blockIdx.y;
    const int b = u / a.num_kv_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = a.rows[b], keep = a.keep[b];
    const size_t at = (static_cast<size_t>(layer) * a.n_seqs + a.b0) * a.num_kv_heads + u;
    const float *w = a.weights + at * a.w_stride;
    int32_t *kept = a.kept + at * a.kept_stride;
    float *w_out = a.weights_out ? a.weights_out + at * a.w_stride : nullptr;
    const bool all = keep >= n;
    const int lo = all ? n : a.first, hi = all ? n : n - a.recent;  // rows to choose from (none: all stay)
    int want = all ? 0 : keep - a.first - a.recent;                 // of those
    auto key_at = [&](int j) -> uint32_t {
        if constexpr (kLds) return keys[j];
        return order_key(w[j]);
    };
    if constexpr (kLds) {
        for (int j = lo + tid; j < hi; j += kSelectThreads) keys[j] = order_key(w[j]);
    }
    // Digits of the least key that stays; `want` counts down to its equals.
    uint32_t prefix = 0;
    int shift = 32;
    if (want > 0) {
#pragma unroll 1
        for (int round = 0; round < 3; ++round) {
            const int bits = round == 0 ? 12 : 10;
            const uint32_t done = shift == 32 ? 0u : ~0u << shift;
            shift -= bits;
            const int bins = 1 << bits;
            for (int i = tid; i < bins; i += kSelectThreads) hist[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += kSelectThreads) {
                const uint32_t k = key_at(j);
                if ((k & done) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
            }
            __syncthreads();
            // Counters from the largest digit down, `per` to a thread.
            const int per = bins / kSelectThreads;  // 4 or 1
            int mine = 0;
            for (int i = 0; i < per; ++i) mine += hist[bins - 1 - (tid * per + i)];
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(upto, o);
                upto += lane >= o ? x : 0;
            }
            if (lane == 63) wave_sum[wave] = upto;
            __syncthreads();
            int before = upto - mine;
            for (int v = 0; v < wave; ++v) before += wave_sum[v];
            if (before < want && want <= before + mine) {  // one thread
                for (int i = 0; i < per; ++i) {
                    const int digit = bins - 1 - (tid * per + i), c = hist[digit];
                    if (want <= before + c) {
                        found[0] = digit;
                        found[1] = before;
                        break;
                    }
                    before += c;
                }
            }
            __syncthreads();
            prefix |= static_cast<uint32_t>(found[0]) << shift;
            want -= found[1];
            __syncthreads();
        }
    } else if constexpr (kLds) {
        __syncthreads();
    }
    // Rows by waves, a run of them each: first the counts, then the places.
    const int j0 = static_cast<int>(static_cast<int64_t>(n) * wave / kSelectWaves);
    const int j1 = static_cast<int>(static_cast<int64_t>(n) * (wave + 1) / kSelectWaves);
    const bool any = !all && keep > a.first + a.recent;
    auto sort_of = [&](int j, bool &stay, bool &tie) {  // row j < j1
        const bool held = j < lo || j >= hi;
        const uint32_t k = !held && any ? key_at(j) : 0u;
        stay = held || (any && k > prefix);
        tie = !held && any && k == prefix;
    };
    int n_stay = 0, n_tie = 0;
    for (int j = j0 + lane; j - lane < j1; j += 64) {
        bool stay = false, tie = false;
        if (j < j1) sort_of(j, stay, tie);
        n_stay += __popcll(__ballot(stay));
        n_tie += __popcll(__ballot(tie));
    }
    if (lane == 0) {
        wave_sum[wave] = n_stay;
        wave_tie[wave] = n_tie;
    }
    __syncthreads();
    int ties = 0, out = 0;
    for (int v = 0; v < wave; ++v) {
        out += wave_sum[v];
        ties += wave_tie[v];
    }
    out += min(ties, want);  // equals that stayed before this run
    const uint64_t below = (1ull << lane) - 1;
    for (int j = j0 + lane; j - lane < j1; j += 64) {
        bool stay = false, tie = false;
        if (j < j1) sort_of(j, stay, tie);
        const uint64_t tie_set = __ballot(tie);
        stay = stay || (tie && ties + __popcll(tie_set & below) < want);
        const uint64_t set = __ballot(stay);
        if (stay) {
            const int i = out + __popcll(set & below);
            kept[i] = j;
            if (w_out) w_out[i] = w[j];
        }
        out += __popcll(set);
        ties += __popcll(tie_set);
    }
    const int m = min(keep, n);
    for (int64_t i = m + tid; i < a.kept_stride; i += kSelectThreads) kept[i] = -1;
    if (w_out)
        for (int64_t i = m + tid; i < a.w_stride; i += kSelectThreads) w_out[i] = 0.0f;
}

// ---- the rows that stay, in pages of their own ----------------------------------

// grid (record, KV head, layer), a half-wave per row of a destination page.
// Nothing that is read is written: destinations are other blocks than the
// sources', and the last page of an 8-bit cache goes to the sequence's other open
// block.
template <bool kInt8>
__global__ __launch_bounds__(32 * kBlockTokens) void gather_kernel(GatherArgs a) {
    __shared__ CloseLds lds;
    const int hkv = gridDim.y, h = blockIdx.y, layer = blockIdx.z;
    const int row = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const int32_t *rec = a.recs + static_cast<size_t>(blockIdx.x) * kTouchWords;
    const int b = ld_uniform(rec), page = ld_uniform(rec + 1), src = ld_uniform(rec + 2), blk = ld_uniform(rec + 3);
    const int n = ld_uniform(rec + 4), src_open = ld_uniform(rec + 5), src_slot = ld_uniform(rec + 6);
    const int32_t *kept = a.kept + ((static_cast<size_t>(layer) * a.n_seqs + b) * hkv + h) * a.kept_stride + 16 * page;
    const int32_t *trow = a.table + static_cast<size_t>(src) * a.table_stride;
    BlockRow x{};
    if constexpr (kInt8) {
        uint8_t *k8 = a.k8 + layer * a.layer_codes, *v8 = a.v8 + layer * a.layer_codes;
        float *scales = a.scales + layer * a.layer_scales;
        uint16_t *open = a.open + layer * a.layer_open;
        if (row < n) {
            const int j = kept[row], pg = j >> 4;
            if (pg == src_open) {
                x = load_open_row(open + (static_cast<size_t>(src_slot) * hkv + h) * 2 * kPageElems, j & 15, l32);
            } else {
                const size_t at = static_cast<size_t>(trow[pg]) * hkv + h;
                x = load_code_row(k8 + at * kPageElems, v8 + at * kPageElems, scales + 2 * at, j & 15, l32);
            }
        }
        if (blk < 0) {  // uniform
            if (row < n) store_open_row(open + (static_cast<size_t>(-1 - blk) * hkv + h) * 2 * kPageElems, row, l32, x);
            return;
        }
        const size_t at = static_cast<size_t>(blk) * hkv + h;
        close_block(x, k8 + at * kPageElems, v8 + at * kPageElems, scales + 2 * at, lds);
    } else {
        if (row >= n) return;
        const int j = kept[row];
        const uint16_t *kp = a.k_pool + layer * a.layer_elems, *vp = a.v_pool + layer * a.layer_elems;
        const size_t from = ((static_cast<size_t>(trow[j >> 4]) * kBlockTokens + (j & 15)) * hkv + h) * kHeadDim + 8 * l32;
        const size_t to = ((static_cast<size_t>(blk) * kBlockTokens + row) * hkv + h) * kHeadDim + 8 * l32;
        x.k = ld16(kp + from);
        x.v = ld16(vp + from);
        st16(a.k_pool + layer * a.layer_elems + to, x.k);
        st16(a.v_pool + layer * a.layer_elems + to, x.v);
    }
}

template <bool kInt8, int NT>
hipError_t launch_weights_tiles(const WeightArgs &a, hipStream_t s) {
    const dim3 grid(a.splits, a.num_kv_heads, a.n_seqs), block(64 * kWeightWaves);
    hipLaunchKernelGGL((stats_kernel<kInt8, NT>), grid, block, 0, s, a);
    hipLaunchKernelGGL((sum_kernel<kInt8, NT>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <bool kInt8>
hipError_t launch_weights_kind(const WeightArgs &a, hipStream_t s) {
    const int tiles = (a.n_obs * (a.num_heads / a.num_kv_heads) + 15) / 16;
    if (tiles <= 1) return launch_weights_tiles<kInt8, 1>(a, s);
    if (tiles <= 4) return launch_weights_tiles<kInt8, 4>(a, s);
    if (tiles <= 8) return launch_weights_tiles<kInt8, 8>(a, s);
    if (tiles <= 16) return launch_weights_tiles<kInt8, 16>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_weights(const WeightArgs &a, hipStream_t s) {
    if (a.n_seqs <= 0) return hipSuccess;
    return a.k8 ? launch_weights_kind<true>(a, s) : launch_weights_kind<false>(a, s);
}

hipError_t launch_select(const SelectArgs &a, int32_t n, int32_t n_layers, int32_t most, hipStream_t s) {
    if (n <= 0) return hipSuccess;
    const dim3 grid(n * a.num_kv_heads, n_layers), block(kSelectThreads);
    if (most <= kSelectLds) {
        const size_t lds = static_cast<size_t>(most) * sizeof(uint32_t);
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(select_kernel<true>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSelectLds * sizeof(uint32_t));
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(select_kernel<true>, grid, block, lds, s, a);
    } else {
        hipLaunchKernelGGL(select_kernel<false>, grid, block, 0, s, a);
    }
    return hipGetLastError();
}

hipError_t launch_gather(const GatherArgs &a, int32_t n_recs, int32_t num_kv_heads, int32_t n_layers, hipStream_t s) {
    if (n_recs <= 0) return hipSuccess;
    const dim3 grid(n_recs, num_kv_heads, n_layers), block(32 * kBlockTokens);
    if (a.k8)
        hipLaunchKernelGGL(gather_kernel<true>, grid, block, 0, s, a);
    else
        hipLaunchKernelGGL(gather_kernel<false>, grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace kva
