// Eviction by accumulated attention weight, over FP16 and 8-bit caches (gfx950):
// what the step's last tokens look at (stats_kernel, sum_kernel), which rows
// stay (select_kernel), and those rows in pages of their own (gather_kernel).
//
// Weights.  For a sequence's last m = min(new tokens, n_obs) tokens and the G
// query heads of a KV head: w[row] = decay * w[row] + sum over (token, head) of
// softmax(q K^T / 16)[row], each token seeing rows up to its own.  Query rows are
// (token, head) pairs, 16 to a tile, the operand B of 16x16x32 products, in LDS
// for the whole workgroup; a wave takes two pages as A and multiplies them with
// every tile, so an operand read from LDS serves two products.  In the C layout
// a lane holds one query row (column l % 16) and four keys of each page (4 (l /
// 16) .. + 3).  A first pass over K leaves every query row's max and sum, which
// stay in the lane until the end; then
//   - up to 16 query rows (a decode step), it leaves the scores too (a query
//     row's are 4 bytes to a key's 256 or 512), and the probabilities are made and
//     summed from them (score_kernel);
//   - more rows, the scores would outweigh the keys, and a second pass over K
//     sums the probabilities, in the lane over its tiles, before the sixteen
//     lanes of a row once per page (sum_kernel).
// A workgroup takes a chunk of a sequence's pages, the same number for every
// sequence, so a ragged batch is shared out by its pages.
//
// A decode step is bound by HBM and by its start (dependent loads: the plan, the
// page ids, the first keys): 32 sequences of 1024 to 8192 rows (5200 in the mean) in
// 8 bits, 171 MB of K, take 42 us in stats_kernel and 8 in score_kernel; a walk of
// equal shares through LDS, as the 8-bit decode's, took 45 in place of the 42.
// Many rows are bound by the vector unit and LDS: four sequences of 9000 to 16000
// rows (13300 in the mean) with 192 query rows, FP16, 40 us and 39 (the products
// alone would take 8).
#include <type_traits>

#include "k_common.h"
#include "k_page8.h"
#include "kva_internal.h"

namespace kva {
namespace {

constexpr float kQkScale = 1.4426950408889634f / 16.0f;

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
// lane's B holds at each k-step: 64 (s / 2) + 16 (l / 16) + 8 (s % 2) .. + 7, the
// order of an 8-bit page; of an FP16 row, two steps take a 128-byte line.
// raw: what memory holds of them.
template <bool kInt8>
struct Keys {
    uint4 raw[kInt8 ? 4 : 8];
    float factor;  // of the scores, log2(e) / 16 included
};
__device__ __forceinline__ int query_dim(int s, int grp) { return 64 * (s >> 1) + 16 * grp + 8 * (s & 1); }

// What a workgroup works on: pages [p0, p1) of sequence b for KV head h; obs:
// query tokens, from token `tok` of the step; slot: the open block; page0: pages
// of earlier sequences; the sequence's chunks are [c0, c1).
struct Span {
    int b, h, sid, slot, ctx, obs, tok, p0, p1, page0, c0, c1;
};
__device__ __forceinline__ Span span_of(const WeightArgs &a) {
    Span s;
    const int lane = threadIdx.x & 63, x = blockIdx.x;
    // The sequence whose chunks hold chunk x: 64 sequences at a time.
    int base = 0, b = 0;
    for (int g = 0; g < a.n_seqs; g += 64) {
        const int i = g + lane;
        int n = i < a.n_seqs ? (a.pre_seq[i + 1] - a.pre_seq[i] + a.chunk - 1) / a.chunk : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(n, o);
            n += lane >= o ? y : 0;
        }
        const uint64_t before = __ballot(base + n <= x);  // sequences that end at or before it: a prefix
        if (before != ~0ull) {
            const int k = __popcll(before);
            s.c0 = base + (k ? __builtin_amdgcn_readlane(n, k - 1) : 0);
            s.c1 = base + __builtin_amdgcn_readlane(n, k);
            b = g + k;
            break;
        }
        base += __builtin_amdgcn_readlane(n, 63);
    }
    s.b = __builtin_amdgcn_readfirstlane(b);
    s.c0 = __builtin_amdgcn_readfirstlane(s.c0);
    s.c1 = __builtin_amdgcn_readfirstlane(s.c1);
    s.h = blockIdx.y;
    s.sid = ld_uniform(a.seq_ids + s.b);
    s.slot = a.k8 ? ld_uniform(a.open_slot + s.b) : 0;
    s.ctx = ld_uniform(a.ctx_lens + s.b);
    s.page0 = ld_uniform(a.pre_seq + s.b);
    const int t0 = ld_uniform(a.tok_off + s.b), t1 = ld_uniform(a.tok_off + s.b + 1);
    s.obs = min(t1 - t0, a.n_obs);
    s.tok = t1 - s.obs;
    s.p0 = (x - s.c0) * a.chunk;
    s.p1 = min(s.p0 + a.chunk, (s.ctx + kBlockTokens - 1) / kBlockTokens);
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
            a.k_pool + ((static_cast<size_t>(id) * kBlockTokens + (lane & 15)) * hkv + s.h) * kHeadDim + 16 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) k.raw[i] = ld16(src + query_dim(i, 0));
        k.factor = kQkScale;
    }
}
template <bool kInt8>
__device__ __forceinline__ void operands(half8_t (&op)[8], const Keys<kInt8> &k) {
    if constexpr (kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            op[2 * i] = as_h8(codes8(k.raw[i].x, k.raw[i].y));
            op[2 * i + 1] = as_h8(codes8(k.raw[i].z, k.raw[i].w));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) op[i] = as_h8(k.raw[i]);
    }
}

// The span's query rows to LDS as B operands: [tile][k-step][lane] of 16 bytes,
// zeros past the last row.  Requested together: a workgroup starts with them.
template <int NT, int WAVES>
__device__ __forceinline__ void load_queries(uint4 *qs, const WeightArgs &a, const Span &s) {
    constexpr int kEach = NT * 512 / (64 * WAVES);
    const int G = a.num_heads / a.num_kv_heads;
    uint4 x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = threadIdx.x + 64 * WAVES * e;
        const int lane = i & 63, step = (i >> 6) & 7, row = 16 * (i >> 9) + (lane & 15);
        const int iq = row / G;
        x[e] = iq < s.obs ? ld16(a.q + (static_cast<size_t>(s.tok + iq) * a.num_heads + s.h * G + row - iq * G) * kHeadDim +
                                 query_dim(step, lane >> 4))
                          : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) qs[threadIdx.x + 64 * WAVES * e] = x[e];
}

// The page ids of a walk, 64 to a vector load, one per lane: as scalar loads
// they would make every wait for LDS a wait for them.  Places only go up.
struct PageIds {
    const int32_t *row;
    int base, ids;
    __device__ __forceinline__ void load(int from, int last, int lane) {
        base = from;
        ids = row[min(from + lane, last)];
        // Taken in here: a load that one path leaves pending would make every
        // later use wait for all loads in flight.
        asm volatile("" : "+v"(ids));
    }
    __device__ __forceinline__ int at(int page, int last, int lane) {
        if (page - base >= 64) load(page, last, lane);  // wave-uniform
        return __builtin_amdgcn_readlane(ids, page - base);
    }
};

// Pages that a wave takes at a time: two share the operands read from LDS; with
// one tile of query rows there is little to share, and more waves fit.
constexpr int pages_for(int tiles) { return tiles == 1 ? 1 : 2; }

// Walks the span's pages, PG at a time, this wave's in turn: scores(t, x, f, seen)
// gets tile t's products with them, f times which are log2 units, with -inf (and f
// = 1) where the row does not see the key or there is no such page; seen(j, i):
// whether the row sees key i of page j, which tells those from a score that is
// -inf (an infinite key or query); done(page) ends them.
template <bool kInt8, int NT, int WAVES, class Scores, class Done>
__device__ __forceinline__ void walk(const WeightArgs &a, const Span &s, const uint4 *qs, Scores scores, Done done) {
    constexpr int PG = pages_for(NT);
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.num_heads / a.num_kv_heads;
    // The open page of an 8-bit cache is FP16 rows and goes by itself, after the others.
    const int end = kInt8 ? min(s.p1, s.ctx / kBlockTokens) : s.p1;
    const int last = end - 1;
    int p = s.p0 + PG * wave;
    half8_t op[PG][8];
    float factor[PG];
    // Every tile of query rows against the pages in op, of which `there` are: masked, or every
    // query row sees every key (rows that there are not have zeros for q, so scores
    // of 0, or of NaN with an infinite key; nothing of them is written or summed).
    auto tiles = [&](int page, int there, auto masked) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float4_t x[PG];
            float f[PG];
            [[maybe_unused]] int see[PG];
#pragma unroll
            for (int j = 0; j < PG; ++j) x[j] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const half8_t b = as_h8(qs[(t * 8 + k) * 64 + lane]);
#pragma unroll
                for (int j = 0; j < PG; ++j) x[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op[j][k], b, x[j], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < PG; ++j) {
                f[j] = factor[j];
                if constexpr (masked) {
                    // The last key that the lane's query row sees (none: no such row).
                    // Divided by here: FP16's keys leave no registers for a quotient per
                    // tile from step to step.
                    int g = G;
                    if constexpr (!kInt8) asm volatile("" : "+s"(g));
                    const int iq = (16 * t + col) / g;
                    see[j] = iq < s.obs && j < there ? s.ctx - s.obs + iq : -1;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[j][i] = 16 * (page + j) + 4 * grp + i <= see[j] ? x[j][i] * factor[j] : -INFINITY;
                    f[j] = 1.0f;
                }
            }
            scores(t, x, f, [&](int j, int i) {
                if constexpr (masked) return 16 * (page + j) + 4 * grp + i <= see[j];
                return 16 * t + col < s.obs * G;
            });
            // Two tiles' reads and products overlap; more would only cost registers.
            if (t & 1) __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (kInt8 && end < s.p1 && wave == WAVES - 1) {
        const uint16_t *src = a.open + (static_cast<size_t>(s.slot) * a.num_kv_heads + s.h) * 2 * kPageElems + 16 * lane;
#pragma unroll
        for (int j = 0; j < PG; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) op[j][i] = as_h8(ld16(src + 1024 * (i >> 1) + 8 * (i & 1)));
            factor[j] = kQkScale;
        }
        tiles(end, 1, std::true_type{});
        done(end);
    }
    if (p > last) return;
    PageIds ids{a.table + static_cast<size_t>(s.sid) * a.table_stride, 0, 0};
    ids.load(p, last, lane);
    Keys<kInt8> keys[2][PG];
    auto request = [&](Keys<kInt8> (&k)[PG], int page) {
#pragma unroll
        for (int j = 0; j < PG; ++j) {
            const int q = min(page + j, last);
            load_keys(k[j], a, s, q, ids.at(q, last, lane), lane);
        }
    };
    request(keys[0], p);
    // One step: the pages in `cur`, with the next step's requested first.  (More
    // steps on their way take longer: 32 sequences of 1000 rows, 8-bit and FP16,
    // 14.1 and 19.9 us with one, 14.4 with three and 21.8 with two; of 8000 the same.)
    auto step = [&](const Keys<kInt8> (&cur)[PG], Keys<kInt8> (&nxt)[PG]) -> bool {
        request(nxt, p + PG * WAVES);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < PG; ++j) {
            operands<kInt8>(op[j], cur[j]);
            factor[j] = cur[j].factor;
        }
        if (p + PG - 1 <= last && 16 * (p + PG) - 1 <= s.ctx - s.obs)
            tiles(p, PG, std::false_type{});
        else
            tiles(p, last - p + 1, std::true_type{});
        done(p);
        p += PG * WAVES;
        return p <= last;
    };
    while (step(keys[0], keys[1]) && step(keys[1], keys[0])) {
    }
}

__device__ __forceinline__ float exp_sum(const float4_t &x, float f, float mu) {
    return (__builtin_amdgcn_exp2f(fmaf(x[0], f, -mu)) + __builtin_amdgcn_exp2f(fmaf(x[1], f, -mu))) +
           (__builtin_amdgcn_exp2f(fmaf(x[2], f, -mu)) + __builtin_amdgcn_exp2f(fmaf(x[3], f, -mu)));
}
__device__ __forceinline__ float max4(const float4_t &x) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); }

// (m, l) of every query row over the chunk: part[chunk][h][row].  kScores: and
// the scores, scores[page of the step][h][row][16 keys] (one tile).
template <bool kInt8, int NT, int WAVES, bool kScores>
__global__ __launch_bounds__(64 * WAVES) void stats_kernel(WeightArgs a) {
    static_assert(!kScores || NT == 1, "one tile of scores");
    __shared__ uint4 qs[NT * 512];
    __shared__ float2 wave_ml[WAVES][NT * 16];
    const Span s = span_of(a);
    if (s.obs == 0) return;
    const int rows = s.obs * (a.num_heads / a.num_kv_heads);
    load_queries<NT, WAVES>(qs, a, s);
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
    }
    constexpr int PG = pages_for(NT);
    float4_t kept = float4_t{0.f, 0.f, 0.f, 0.f};
    walk<kInt8, NT, WAVES>(
        a, s, qs,
        [&](int t, const float4_t (&x)[PG], const float (&f)[PG], auto) {
            float mn = m[t], sum = 0.0f;
#pragma unroll
            for (int j = 0; j < PG; ++j) mn = fmaxf(mn, max4(x[j]) * f[j]);  // f >= 0 keeps the order
            const float mu = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
            for (int j = 0; j < PG; ++j) sum += exp_sum(x[j], f[j], mu);
            l[t] = l[t] * __builtin_amdgcn_exp2f(m[t] - mu) + sum;
            m[t] = mn;
            if constexpr (kScores) kept = x[0] * f[0];
        },
        [&](int page) {
            if constexpr (kScores) {
                const int col = lane & 15, grp = lane >> 4;
                const size_t at = (static_cast<size_t>(s.page0 + page) * a.num_kv_heads + s.h) * a.part_rows;
                if (col < rows) *reinterpret_cast<float4_t *>(a.scores + (at + col) * kBlockTokens + 4 * grp) = kept;
            }
        });
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float mx = group4_max(m[t]);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float lt = group4_sum(l[t] * __builtin_amdgcn_exp2f(m[t] - mu));
        if (lane < 16) wave_ml[wave][16 * t + lane] = make_float2(mx, lt);
    }
    __syncthreads();
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
        float mx = -INFINITY, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, wave_ml[w][r].x);
        const float mu = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) lt += wave_ml[w][r].y * __builtin_amdgcn_exp2f(wave_ml[w][r].x - mu);
        a.part[(static_cast<size_t>(blockIdx.x) * a.num_kv_heads + s.h) * a.part_rows + r] = make_float2(mx, lt);
    }
}

// A query row's max and 1 / sum over the sequence's chunks, by 16 lanes of a
// DPP row: row r of rows rows by the lanes that hold r, every lane gets them.
// Rows that there are not weigh nothing.  `first` is the lane's first partial,
// requested before (a workgroup starts with these).
__device__ __forceinline__ float2 first_part(const WeightArgs &a, const Span &s, int r, int rows, int l16) {
    if (r >= rows || l16 >= s.c1 - s.c0) return make_float2(-INFINITY, 0.0f);
    return a.part[(static_cast<size_t>(s.c0 + l16) * a.num_kv_heads + s.h) * a.part_rows + r];
}
// (max, 1 / sum) of the (max, sum) of a DPP row's 16 lanes.
__device__ __forceinline__ float2 row_merge(float mx, float lt) {
    float all = mx;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
    const float mu = all == -INFINITY ? 0.0f : all;
    return make_float2(mu, 1.0f / row16_sum(lt * __builtin_amdgcn_exp2f(mx - mu)));
}
__device__ __forceinline__ float2 row_stat(const WeightArgs &a, const Span &s, float2 first, int r, int rows, int l16) {
    float mx = first.x, lt = first.y;
    if (r < rows)
        for (int i = s.c0 + l16 + 16; i < s.c1; i += 16) {
            const float2 p = a.part[(static_cast<size_t>(i) * a.num_kv_heads + s.h) * a.part_rows + r];
            const float mn = fmaxf(mx, p.x);
            const float mu = mn == -INFINITY ? 0.0f : mn;
            lt = lt * __builtin_amdgcn_exp2f(mx - mu) + p.y * __builtin_amdgcn_exp2f(p.x - mu);
            mx = mn;
        }
    const float2 all = row_merge(mx, lt);
    return r < rows ? all : make_float2(0.0f, 0.0f);
}

__device__ __forceinline__ void put_weight(const WeightArgs &a, const Span &s, int key, float x) {
    float *w = a.weights + (static_cast<size_t>(s.b) * a.num_kv_heads + s.h) * a.w_stride + key;
    *w = a.decay == 0.0f ? x : fmaf(a.decay, *w, x);
}

// The probabilities of the chunk's rows, summed over the query rows, onto the
// decayed weights: from K.
template <bool kInt8, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void sum_kernel(WeightArgs a) {
    __shared__ uint4 qs[NT * 512];
    __shared__ float2 stat[NT * 16];
    const Span s = span_of(a);
    const int rows = s.obs * (a.num_heads / a.num_kv_heads);
    if (s.obs == 0) {  // decayed only
        for (int key = 16 * s.p0 + threadIdx.x; key < min(16 * s.p1, s.ctx); key += blockDim.x) put_weight(a, s, key, 0.0f);
        return;
    }
    constexpr int kEach = NT * 256 / (64 * WAVES);
    float2 first[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) first[e] = first_part(a, s, 4 * WAVES * e + (threadIdx.x >> 4), rows, threadIdx.x & 15);
    load_queries<NT, WAVES>(qs, a, s);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int r = 4 * WAVES * e + (threadIdx.x >> 4);
        const float2 x = row_stat(a, s, first[e], r, rows, threadIdx.x & 15);
        if ((threadIdx.x & 15) == 0) stat[r] = x;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    constexpr int PG = pages_for(NT);
    const int end = kInt8 ? min(s.p1, s.ctx / kBlockTokens) : s.p1;  // full pages
    float4_t sum[PG] = {};
    walk<kInt8, NT, WAVES>(
        a, s, qs,
        [&](int t, const float4_t (&x)[PG], const float (&f)[PG], auto seen) {
            const float2 st = stat[16 * t + col];
#pragma unroll
            for (int j = 0; j < PG; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(x[j][i], f[j], -st.x));
                    // A row that does not see the key (p = 0) adds nothing, whatever
                    // its sum is; one that does adds NaN where its sum is NaN or zero
                    // (none but scores of -inf), also at p = 0.
                    const float y = fmaf(p, st.y, sum[j][i]);
                    sum[j][i] = seen(j, i) ? y : sum[j][i];
                }
        },
        [&](int page) {
#pragma unroll
            for (int j = 0; j < PG; ++j) {
                float mine = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float all = row16_sum(sum[j][i]);
                    mine = col == i ? all : mine;
                }
                sum[j] = float4_t{0.f, 0.f, 0.f, 0.f};
                const int key = 16 * (page + j) + 4 * grp + col;
                if (col < 4 && (j == 0 || page + j < end) && key < s.ctx) put_weight(a, s, key, mine);
            }
        });
}

// The same from the scores that stats_kernel left: a thread per key.
__global__ __launch_bounds__(256) void score_kernel(WeightArgs a) {
    __shared__ float2 stat[16];
    __shared__ int last[16];  // the last key that the row sees
    const Span s = span_of(a);
    const int G = a.num_heads / a.num_kv_heads;
    const int rows = s.obs * G;  // at most 16
    const int r0 = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int end = min(16 * s.p1, s.ctx);
    float *w = a.weights + (static_cast<size_t>(s.b) * a.num_kv_heads + s.h) * a.w_stride;
    float v[16], old = 0.0f;
    auto request = [&](int key) {
        if (a.decay != 0.0f) old = w[key];
        const float *x = a.scores +
                         (static_cast<size_t>(s.page0 + (key >> 4)) * a.num_kv_heads + s.h) * a.part_rows * kBlockTokens +
                         (key & 15);
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = r < rows ? x[r * kBlockTokens] : -INFINITY;
    };
    int key = 16 * s.p0 + threadIdx.x;
    const float2 first = first_part(a, s, r0, rows, l16);
    if (key < end) request(key);
    const float2 mine = row_stat(a, s, first, r0, rows, l16);
    if (l16 == 0) {
        stat[r0] = mine;
        last[r0] = r0 < rows ? s.ctx - s.obs + r0 / G : -1;
    }
    __syncthreads();
    while (key < end) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (key <= last[r]) sum += __builtin_amdgcn_exp2f(v[r] - stat[r].x) * stat[r].y;
        w[key] = fmaf(a.decay, old, sum);
        key += blockDim.x;
        if (key < end) request(key);
    }
}

// ---- which rows stay ---------------------------------------------------------

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// Larger weights have larger keys; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w == w ? w + 0.0f : -INFINITY);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// Whether the weight is its key's value, bit for bit.
__device__ __forceinline__ bool key_tells(uint32_t key) { return key != ~0xff800000u && key != 0x80000000u; }
__device__ __forceinline__ float key_value(uint32_t key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// A workgroup per (sequence and KV head, layer).  The key of the last row that
// stays is found by its digits (12, 10 and 10 bits, the first with sign, exponent
// and three bits of the significand, so that weights of a few binades spread
// over many counters); then the rows above it, and as many of its equals from
// the lowest place on as there is room for, are written in order.  kLds: the
// keys are held in LDS (up to kSelectLds rows), else read again for each step.
// The weights are few (64 KB of 16384 rows); the time goes by in waits, so they
// are requested eight to a thread, and those that stay are written from their
// keys (16384 rows, 2048 of them kept: 28 us; one at a time and read again 32).
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
        constexpr int kEach = 8;
        for (int j0 = tid; j0 < n; j0 += kEach * kSelectThreads) {
            float x[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) x[i] = w[min(j0 + i * kSelectThreads, n - 1)];
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (j0 + i * kSelectThreads < n) keys[j0 + i * kSelectThreads] = order_key(x[i]);
        }
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
            if (w_out) w_out[i] = kLds && key_tells(keys[j]) ? key_value(keys[j]) : w[j];
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

// grid (record, KV head, layer), a half-wave per row of a destination page.  Bound
// by memory: 200 MB of FP16 rows read here and there and written in order 79 us,
// 5.1 TB/s.  The same rows of an 8-bit cache, half the bytes, take 119 us: a row's
// codes lie among those of its block's other rows (K's in pieces of 16 bytes, V's
// one by one), so 100 MB of them fetch two to four times that, in loads of 8
// bytes and of one.
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

template <bool kInt8, int NT, int WAVES>
hipError_t launch_weights_tiles(const WeightArgs &a, hipStream_t s) {
    const dim3 grid(a.n_chunks, a.num_kv_heads), block(64 * WAVES);
    if constexpr (NT == 1) {
        if (a.scores) {
            hipLaunchKernelGGL((stats_kernel<kInt8, 1, WAVES, true>), grid, block, 0, s, a);
            hipLaunchKernelGGL(score_kernel, grid, dim3(256), 0, s, a);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((stats_kernel<kInt8, NT, WAVES, false>), grid, block, 0, s, a);
    hipLaunchKernelGGL((sum_kernel<kInt8, NT, WAVES>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <bool kInt8>
hipError_t launch_weights_kind(const WeightArgs &a, hipStream_t s) {
    switch (weight_tiles(a.part_rows)) {
        case 1: return launch_weights_tiles<kInt8, 1, 4>(a, s);
        case 2: return launch_weights_tiles<kInt8, 2, 4>(a, s);
        case 4: return launch_weights_tiles<kInt8, 4, 4>(a, s);
        case 8: return launch_weights_tiles<kInt8, 8, 8>(a, s);
        case 12: return launch_weights_tiles<kInt8, 12, 8>(a, s);
        case 16: return launch_weights_tiles<kInt8, 16, 8>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_weights(const WeightArgs &a, hipStream_t s) {
    if (a.n_chunks <= 0) return hipSuccess;  // no sequence has rows
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
