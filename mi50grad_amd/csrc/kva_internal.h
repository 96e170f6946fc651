// Internal interface between the host side of libkvattn (kva_host.cpp, built
// with g++) and the HIP kernels (k_*.hip, built with hipcc for gfx950).
// Only plain types cross this boundary: fp16 tensors are uint16_t pointers.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace kva {

constexpr int kHeadDim = 256;     // the only head_dim the paged kernels take
constexpr int kBlockTokens = 16;  // tokens per page
constexpr int kDecodeHeadsPerWg = 4;  // kv heads per stream-K decode workgroup (one wave each), at most
constexpr int kSplitQuantum = 16; // decode split sizes are whole pages
constexpr int kCombineRecs = 64;  // sequences whose combine facts travel in the decode arguments
constexpr int kPlanPages = 64;    // page ids per sequence in the step plan (one per lane)
constexpr int kCombineChunk = 16; // decode partials a combine wave requests together
constexpr size_t kPageElems = kBlockTokens * kHeadDim;  // values of a block: a KV head's share of a page, K or V
// A touch: the rows of one page that a step writes.  int32 words: sequence, page
// of it, first row's place among the step's tokens, first row within the page,
// rows, the open block that the page's earlier rows are in or its rows stay in;
// two spare.
constexpr int kTouchWords = 8;

// Fused QK-RMSNorm + RoPE + K/V append over all new tokens of a step.
struct AppendArgs {
    uint16_t *q;              // [T][H][256], normalised + rotated in place
    uint16_t *k;              // [T][Hkv][256], normalised + rotated in place
    const uint16_t *v;        // [T][Hkv][256]
    const uint16_t *q_w;      // [256]
    const uint16_t *k_w;      // [256]
    const uint16_t *cos_tab;  // [rows][half_rot]
    const uint16_t *sin_tab;
    uint16_t *k_pool;         // this layer's pool [blocks][16][Hkv][256]
    uint16_t *v_pool;
    const int32_t *table;     // [max_seqs][table_stride]
    int32_t table_stride;
    const int32_t *tok_seq;   // device: sequence id of each new token
    const int32_t *tok_slot;  // device: logical slot of each new token
    const int32_t *tok_pos;   // device: RoPE position of each new token
    int32_t n_tok;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t half_rot;
    float eps;
    int32_t keep_k;           // 1: k is read only (the cache gets the normalised rows)
};
hipError_t launch_append(const AppendArgs &a, hipStream_t s);

// Q/K/V projection of a step's tokens fused with norm + RoPE + K/V append.
// Weight rows: w_a = [Q heads | Q_gate heads] (n_a = 2*H*256 rows), w_b =
// [K heads | V heads] (n_b = 2*Hkv*256 rows), each row `hidden` fp16.  Up to
// 32 tokens of the hidden sizes that fit it stream the weights past x held
// in registers (proj_lds_kernel); everything else runs as LDS-tiled GEMMs
// (k_gemm.hip).  A form that splits hidden among workgroups writes fp32
// partials, and a finish kernel sums them in split order, rounds to fp16
// (the projection the reference's GEMV stores) and finishes each head; an
// unsplit GEMM does that in its own epilogue.
constexpr int kProjTokens = 64;     // tokens the workspace refusals are counted in
constexpr int kProjMaxSplits = 4;   // hidden split among workgroups, at most (proj_lds_kernel)
constexpr int kGemmMaxSplits = 8;   // the same of the GEMM forms
constexpr size_t kProjPartFactor = 4;  // partial workspace over kProjMaxSplits x kProjTokens tokens of every row, at most
constexpr int kProjWaves = 8;       // waves per workgroup
constexpr int kProjRowTiles = 7;    // 16-row weight tiles per workgroup
constexpr int kProjHiddenQuantum = 512;  // hidden must be a multiple of this
constexpr int kProjWgPerCu = 1;     // workgroups per CU the split aims for, at most
constexpr int kProjStreamTokens = 32; // most tokens of the x-resident form
constexpr int kProjStreamSteps = 10;  // its k-steps per wave
constexpr int kProjLdsDepth = 6;      // two-step LDS stages in flight per wave there
// The same form over 6 k-steps per wave (hidden 6144 at four splits: the
// O-projection from 24 heads), with 5 row tiles per workgroup so that 5120
// output rows still make 256 workgroups.
constexpr int kProjStreamStepsB = 6;
constexpr int kProjRowTilesB = 5;
struct ProjectArgs {
    const uint16_t *x;        // [n_tok][hidden]
    const uint16_t *w_a;
    const uint16_t *w_b;
    int32_t n_a, n_b;
    int32_t hidden;
    int32_t n_tok;
    int32_t splits;           // of hidden among workgroups
    // An output overlaps x or a weight: the product goes to partials whole,
    // so that every operand has been read when the finish kernel writes.
    bool hold;
    float *part;              // [splits][n_tok][n_a + n_b]
    uint16_t *q_out;          // [T][H][256]: normalised + rotated Q
    uint16_t *gate_out;       // [T][H][256]: Q_gate as projected (nullable)
    uint16_t *kv_out;         // [T][2][Hkv][256]: K, V as projected (nullable)
    const uint16_t *q_w;
    const uint16_t *k_w;
    const uint16_t *cos_tab;
    const uint16_t *sin_tab;
    uint16_t *k_pool;
    uint16_t *v_pool;
    const int32_t *table;
    int32_t table_stride;
    const int32_t *tok_seq;
    const int32_t *tok_slot;
    const int32_t *tok_pos;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t half_rot;
    float eps;
    // Output projection (launch_out_project; w_a = W_o, n_b = 0): y_out =
    // fp16(x W_o^T + residual), both [T][n_a]; residual nullable, may be y_out.
    uint16_t *y_out;
    const uint16_t *residual;
    // Events around the product's launch (null: none), as in
    // DecodeArgs.
    hipEvent_t ev_before, ev_after;
};
// How gemm_pair_kernel cuts its row tiles.
struct GemmPair {
    int tall, all;         // workgroups of tall tiles, and of both
    int heads;             // row tiles of the first kind
    int hi, lo;            // tall tiles of one row tile of the first kind, of the others
    int rest_hi, rest_lo;  // the same of the low ones
};
// How a product runs: the x-resident form (stream), a tile GEMM or one of two
// tile heights (pair).  Partial: it leaves `splits` partials for a finish
// kernel; else the outputs are written.
struct ProductPlan {
    bool stream, partial;
    int splits;
    int form, pair;   // of the tables in k_gemm.hip (-1: none)
    GemmPair cut;
    int bm, bn, low;  // tile tokens and rows (0 with stream), tokens of the low tiles (0: one height)
};
// The plan of `a`: heads, the Q/K/V projection, else the O-projection.
// `a.splits` is the split of the x-resident form; part_floats what a.part
// holds (the GEMM forms choose their own split from it and the CU count).
// False where no form takes it.
bool plan_product(const ProjectArgs &a, bool heads, int n_cu, size_t part_floats, ProductPlan &plan);
hipError_t launch_project(ProjectArgs a, const ProductPlan &plan, hipStream_t s);
hipError_t launch_out_project(ProjectArgs a, const ProductPlan &plan, hipStream_t s);
// The LDS-tiled GEMMs of both (k_gemm.hip).  Need hidden % 64 == 0.
constexpr int kBigProjMaxTokens = 1 << 24;
bool plan_gemm(const ProjectArgs &a, bool heads, int n_cu, size_t part_floats, ProductPlan &plan);
hipError_t launch_gemm_project(const ProjectArgs &a, bool heads, const ProductPlan &plan, hipStream_t s);
// The finish kernels alone: a.part holds a.splits partials.  once: Q and K are
// rounded only after norm and RoPE.
hipError_t launch_project_finish(const ProjectArgs &a, bool once, hipStream_t s);
hipError_t launch_out_finish(const ProjectArgs &a, hipStream_t s);

// ---- microscaled rows and products (k_mx.hip, k_mxgemm.hip) ----

constexpr int kMxBlock = 32;          // elements of a scale
constexpr int kMxWeightTile = 32;     // rows of a packed weight's tile
constexpr int kMxStreamTokens = 32;   // most tokens of the form that streams the weights past them
constexpr int kMxMaxRows = 1 << 20;   // rows of an output projection's weight, at most (a tile's offsets have 31 bits)
// Values of a call, at most: a launch counts its lanes, eight values each, in 32
// bits.  And values between the first row and the last.
constexpr int64_t kMxMaxValues = int64_t{1} << 34, kMxMaxSpan = int64_t{1} << 40;
constexpr int kMxNormMax = 32768;     // values of a normalised row, at most
struct MxRows {
    const uint16_t *x;        // quantize: [rows] of x_stride values
    int64_t x_stride;
    int64_t rows;
    int32_t cols;
    uint8_t *codes;           // [rows][cols * bits / 8]
    uint8_t *scales;          // [rows][cols / 32]
    uint16_t *y;              // dequantize: [rows][cols]
};
hipError_t launch_mx_quantize(const MxRows &a, int bits, hipStream_t s);
hipError_t launch_mx_dequantize(const MxRows &a, int bits, hipStream_t s);
// A packed weight: codes [row tiles][cols / 64][64 lanes][16], then scales
// [row tiles][cols / 256][64 lanes][4]: of lane l, row l % 32 of the tile, block
// l / 32 of each step of 64; the dword has the bytes of four steps.
struct MxPack {
    const uint8_t *codes, *scales;  // 4-bit rows
    int64_t rows, n_tiles;
    int32_t cols;
    uint8_t *packed;
};
hipError_t launch_mx_pack(const MxPack &a, hipStream_t s);
struct MxNorm {
    const uint16_t *hidden;   // [n_tok][cols]
    const uint16_t *delta;    // nullable
    uint16_t *sum_out;        // hidden + delta (with delta)
    const uint16_t *w;        // [cols]
    void *out;                // fp16 or codes
    uint8_t *scales;
    int32_t n_tok, cols;
    float eps;
};
hipError_t launch_add_rmsnorm(const MxNorm &a, int bits, hipStream_t s);
// The operands of a product by packed weights, beside ProjectArgs' outputs
// (its x, w_a and w_b are not used; hidden, n_a, n_b and n_tok are).
struct MxProduct {
    const uint8_t *x, *x_scales;
    const uint8_t *w_a, *w_b; // packed
    int32_t bits;             // of x
    bool by_kind;             // the order of a tile kernel's heads
};
bool plan_mx(const ProjectArgs &a, const MxProduct &m, bool heads, int n_cu, size_t part_floats, ProductPlan &plan);
hipError_t launch_mx_product(const ProjectArgs &a, const MxProduct &m, bool heads, int n_cu, const ProductPlan &plan,
                             hipStream_t s);

// Reference-compatible norm+RoPE on a contiguous [n_heads][head_dim] buffer.
struct LegacyNormArgs {
    uint16_t *x;
    const uint16_t *w;
    const uint16_t *cos_row;
    const uint16_t *sin_row;
    uint16_t *cache_dst;      // nullable
    int32_t num_heads;
    int32_t head_dim;         // 64, 128 or 256
    int32_t half_rot;
    float eps;
};
hipError_t launch_legacy_norm(const LegacyNormArgs &a, hipStream_t s);

// Split-K GQA decode over a paged (or contiguous) cache.
struct DecodeArgs {
    const uint16_t *q;        // [n_seqs][H][256]
    const uint16_t *k_pool;   // layer base (or contiguous K when table == null)
    const uint16_t *v_pool;
    const int32_t *table;     // device block table, null = contiguous cache
    int32_t table_stride;
    size_t seq_stride;        // contiguous cache: elements between sequences
    const int32_t *seq_ids;   // device [n_seqs] (ignored when table == null)
    const int32_t *ctx_lens;  // device [n_seqs] (null: use ctx_len_const)
    const int32_t *pre_seq;   // device [n_seqs+1]: pages of earlier sequences
                              // (null: every sequence has ctx_len_const)
    // Device [n_seqs][kPlanPages] (null: read the table): the block ids of
    // each sequence's first kPlanPages pages, copied from the table into the
    // step plan when the step began (zeros past its pages), so the
    // whole-sequence form reads them with the length instead of after the
    // sequence id.
    const int32_t *plan_pages;
    int32_t ctx_len_const;
    int32_t n_seqs;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t total_pages;      // pages of all sequences (one page = 16 token rows)
    int32_t n_wg;             // workgroups sharing the pages (stream-K)
    // dyn = 1 (a launch recorded into a replayable graph): total_pages is
    // read from pre_seq[n_seqs] on the device and the workgroup count derived
    // there from split_tokens / min_pages, with n_wg as the cap (the grid).
    int32_t dyn;
    int32_t split_tokens;     // 0 = one workgroup per CU up to the cap
    int32_t min_pages;
    // 1: the host has shown that no sequence is cut into more than
    // kCombineChunk pieces (combine_kernel; else combine_wide_kernel).
    int32_t few_pieces;
    // The combine's view of each sequence, in the kernel arguments so its
    // first loads are the partials (n_crec = n_seqs <= kCombineRecs; 0: it
    // reads the length from the step plan and derives these): crec[b] = the
    // workgroup of the sequence's first piece, -1 when one workgroup covered
    // it; crec_n[b] = 2 * pieces + 1 if the first piece's slot is 2*w0 + 1.
    int32_t n_crec;
    int32_t crec[kCombineRecs];
    int32_t crec_n[kCombineRecs];
    float *ws_acc;            // [2*n_wg][Hkv][G][256] partial slots
    float *ws_ml;             // [2*n_wg][Hkv][G][2]
    uint16_t *out;            // [n_seqs][H][256]
    // Output gate (null = none): out = fp16(fp16(attn) * sigmoid(gate)), the
    // gate row of sequence b, query head hq at gate + b*gate_stride + hq*256.
    const uint16_t *gate;
    int64_t gate_stride;
    int32_t gate_once;        // 1: out = fp16(attn * sigmoid(gate)) (8-bit caches)
    // Per-workgroup timeline (null = off): record kTimelineWords words per
    // wave, [n_wg][grid rows][8 waves], see kva_timeline_read.
    uint64_t *timeline;
    // > 0: whole-sequence form, one workgroup per (sequence, kv head, group
    // of G / whole query heads): no partials, no combine; the stream-K
    // fields are unused.  G / whole must be 1, 2, 3, 4, 6 or 8.
    int32_t whole;
    // Events recorded on the stream right before and after the decode
    // kernel itself (null: none): the dominant kernel's own duration.
    hipEvent_t ev_before, ev_after;
    // 1 (whole form only): the step's append is done in the same launch
    // from `app` (one new token per sequence, token b of sequence b): each
    // workgroup normalises and rotates its query rows (written back in
    // place, q = app.q) and its kv head's new K row, the first group of each
    // (sequence, kv head) writes the new K and V rows to the cache, and the
    // new token joins the attention from registers, not from the cache.
    int32_t fused;
    AppendArgs app;
};
constexpr int kTimelineWords = 4;
constexpr int kWholeWaves = 8;  // waves per whole-sequence decode workgroup
hipError_t launch_decode(const DecodeArgs &a, hipStream_t s);
// The merge of a stream-K launch's partials by itself.
hipError_t launch_decode_merge(const DecodeArgs &a, hipStream_t s);

// Static device scratch of kva_legacy_decode_noalloc (k_noalloc.hip): the
// decode partial slots [2*n_wg][H][256] floats, then [2*n_wg][H][2].
constexpr size_t kNoAllocScratchBytes = size_t(16) << 20;
constexpr int kNoAllocMaxHeads = 128;  // query heads it serves, at most
// The current device's scratch address (fetched once per device with
// hipGetSymbolAddress) and its CU count.
hipError_t noalloc_scratch(void **ptr, int *n_cu);

// Apply block-table patches (seq, index, block) staged by a step.
hipError_t launch_table_patch(int32_t *table, int32_t table_stride,
                              const int32_t *patches, int32_t n_patches,
                              hipStream_t s);

// Streaming device copy (bytes multiple of 16): the HBM bandwidth probe.
hipError_t launch_copy(void *dst, const void *src, size_t bytes, hipStream_t s);
// Read-only stream over `bytes` (multiple of 16): the read-bandwidth probe.
// sink: one word, written only when the data's XOR fold hits a fixed value.
hipError_t launch_read(const void *src, size_t bytes, uint32_t *sink, hipStream_t s);
// Paged read probe: the pages page_ids[0 .. n_pages) (device array) of the
// K and V pools, [page][16][num_kv_heads][256] fp16, read with the stream-K
// decode's per-wave pattern by n_wg workgroups of one wave per kv head.
hipError_t launch_read_pages(const void *k_pool, const void *v_pool, const int32_t *page_ids, int32_t n_pages,
                             int32_t num_kv_heads, int32_t n_wg, uint32_t *sink, hipStream_t s);

// Move accepted rows of each sequence, in every layer (tree rollback).
struct RollbackArgs {
    uint16_t *k_pools;        // base of layer 0; layers are layer_elems apart
    uint16_t *v_pools;
    size_t layer_elems;
    int32_t n_layers;
    const int32_t *table;
    int32_t table_stride;
    const int32_t *moves;     // device [n_moves][3]: seq, src slot, dst slot
    const int32_t *move_off;  // device [n_groups+1]: moves of one sequence
    int32_t n_groups;
    int32_t num_kv_heads;
};
hipError_t launch_rollback(const RollbackArgs &a, hipStream_t s);

// Multi-query (prefill / tree) attention with MFMA tiles.
struct MultiQueryArgs {
    const uint16_t *q;        // [T][H][256]
    uint16_t *out;            // [T][H][256]
    const uint16_t *k_pool;
    const uint16_t *v_pool;
    const int32_t *table;
    int32_t table_stride;
    const int32_t *seq_ids;   // device [n_seqs]
    const int32_t *ctx_lens;  // device [n_seqs]: length after the step
    const int32_t *new_start; // device [n_seqs]: first new slot
    const int32_t *tok_off;   // device [n_seqs+1]: new-token ranges
    const uint64_t *tok_bits; // device [T] (tree mode) or null
    const int32_t *upre;      // device [n_seqs+1]: tiles of earlier sequences (units of one head)
    const int32_t *mq_pre;    // device [n_units+1]: positions of earlier units (blocks + kMqUnitCost each)
    // Device [n_cut][kMqCutWords]: the units cut across workgroups, as
    // kva_step_begin found them from the shares of n_wg (head, first new
    // token of the tile, its valid tokens, first and last share, first
    // piece's slot); the combine launch has one row of workgroups per cut unit.
    const int32_t *mq_cut;
    int32_t n_cut;
    int32_t n_seqs;
    int32_t n_units;          // (kv head, sequence, token tile) units, head-major
    int32_t total_blocks;     // positions of all units (blocks + kMqUnitCost each)
    int32_t keys;             // keys per block: mq_keys_for(n_waves, the step has tree bits)
    int32_t n_wg;             // workgroups sharing the blocks (stream-K)
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t tree;             // 0 = causal chunk, 1 = tree mask
    int32_t n_waves;          // waves per workgroup (4 or 8)
    int32_t n_t;              // 16-row MFMA tiles per wave (1 or 2: mq_two_tiles)
    int32_t q_tile;           // new tokens per unit tile: mq_tile_tokens(G, n_waves, n_t)
    float *ws_acc;            // [2*n_wg][16*n_waves*n_t][256] partial slots
    float *ws_ml;             // [2*n_wg][16*n_waves*n_t][2]
    // Output gate (null = none), as in DecodeArgs: new token t's row of
    // query head hq at gate + t*gate_stride + hq*256.
    const uint16_t *gate;
    int64_t gate_stride;
    // Events around mq_kernel itself (null: none), as in DecodeArgs.
    hipEvent_t ev_before, ev_after;
    // 8-bit cache (k8 null: FP16): this layer's codes, scales and open blocks,
    // as in Store8Args.
    const uint8_t *k8, *v8;
    const float *scales;
    const uint16_t *open;
    const int32_t *open_slot;  // device [n_seqs]
};
// Keys per multi-query block.  64 for a step of eight-wave prefill tiles
// (half the barriers, page lookups and softmax reductions per key, two LDS
// stages of 66 KB: config 4 115.5 -> 110.4 us per call); 32 otherwise, a
// four-stage ring that keeps 96 KB in flight for the HBM-bound tree verify
// (config 5 at 64 keys: 862 -> 888 us) and for small steps.  A step planned
// with tree bits uses 32 for kva_prefill too.
constexpr int mq_keys_for(int waves, bool tree_plan) { return (waves == 8 && !tree_plan) ? 64 : 32; }
// The stream-K split of the multi-query kernel counts each unit as this many
// blocks more than it has: the cost of starting and ending a unit (its query
// rows, its gate and output), so a share full of short units gets fewer
// blocks.  Unit u's blocks sit at positions [mq_pre[u] + cost, mq_pre[u+1]).
// Counted as 2, 3, 4, 5 and 6 blocks, append and attention of a layer: 4 x 512
// tokens after up to 2048 rows 177, 168, 164, 162 and 163 us; 2048 from empty
// 145, 137, 136, 137 and 139, after 16400 rows 900, 900, 881, 887 and 885; 16 x
// 128 from empty 79, 80, 73, 73 and 73; 2 x 1000 after 3000 266, 262, 262, 266
// and 267; in blocks of 32 keys (trees) 64 of nine nodes on up to 1000 rows 165,
// 165, 161, 161 and 164, 8 on up to 3000 52.8, 52.4, 51.4, 51.9 and 52.0.  Of
// sixteen such shapes four is within 2 % of the best on each.
constexpr int kMqUnitCost = 4;
// KV heads (one wave each) of a workgroup of the page walks: the largest divisor
// of all that is at most kDecodeHeadsPerWg.
constexpr int heads_per_wg(int num_kv_heads) {
    int h = num_kv_heads <= kDecodeHeadsPerWg ? num_kv_heads : kDecodeHeadsPerWg;
    while (num_kv_heads % h) --h;
    return h;
}
constexpr int kMqMaxGroup = 8;    // largest GQA group of the multi-query kernel
constexpr int kMqCutWords = 8;    // int32 words of a cut-unit record (6 used)
// Workgroups of a multi-query launch over `blocks` positions: one per CU (the
// cap), at least 128 keys' blocks each.  kva_step_begin (the cut-unit
// records) and the launch must agree.
inline int32_t mq_wg_count(int64_t blocks, int32_t keys, int32_t cap) {
    const int64_t min_blocks = 128 / keys;
    const int64_t w = (blocks + min_blocks - 1) / min_blocks;
    return static_cast<int32_t>(w < 1 || cap < 1 ? 1 : (w > cap ? cap : w));
}
// First position of share w of W over n positions (the device's mq_wg_start).
inline int32_t mq_share_start(int64_t w, int64_t n, int64_t W) { return static_cast<int32_t>(w * n / W); }
// A unit's query rows are (token, head) pairs of the GQA group, 16 per
// MFMA tile, n_t tiles per wave: tokens per unit tile.
constexpr int mq_tile_tokens(int G, int n_waves, int n_t) { return 16 * n_waves * n_t / G; }
// Waves for a step whose longest new-token run is max_new: four (one per
// SIMD) when a whole run fits one unit of 64 rows (tree verify), else eight
// (128 rows; two waves per SIMD hide each other's softmax and LDS waits).
constexpr int mq_waves_for(int G, int max_new) { return max_new * G <= 64 ? 4 : 8; }
// Whether an eight-wave causal step takes two row tiles per wave: with
// `blocks` 64-key blocks in one-tile units over `wgs` workgroups.  Two tiles
// save 15 % of a block's time and cost about 13 us in partials and unit
// starts: 2048 tokens after 16400 rows (417 blocks a workgroup) 778 + 28 us
// of combine against 955 + 19, after 4000 (120) 272 + 28 against 308 + 18;
// 512 after 4000 (26) 83 + 15 against 80 + 11.
constexpr bool mq_two_tiles(int64_t blocks, int32_t wgs) { return blocks >= 48 * static_cast<int64_t>(wgs); }
hipError_t launch_multi_query(const MultiQueryArgs &a, hipStream_t s);

// ---- the 8-bit cache (page order, scales, codes: k_page8.h) ----

// Append into an 8-bit cache.  norm: ap.q and ap.k as in launch_append; else
// ap.k and ap.v are rows as the cache takes them, and ap.q is not touched.
struct Store8Args {
    AppendArgs ap;
    const int32_t *touch;     // device [n_touch][kTouchWords]
    int32_t n_touch;
    int32_t norm;
    uint8_t *k8, *v8;         // this layer's codes [blocks][Hkv][kPageElems]
    float *scales;            // [blocks][Hkv][2]: K's, V's
    uint16_t *open;           // open blocks [max_seqs * 2][Hkv][2: K, V][kPageElems]
};
hipError_t launch_store8(const Store8Args &a, hipStream_t s);
// append_rows on an FP16 cache: ap.k, ap.v to their slots as they are.
hipError_t launch_copy_rows(const AppendArgs &a, hipStream_t s);
// Decode over an 8-bit cache: d as in launch_decode, on its paged stream-K
// path, but for the pools.
struct Decode8Args {
    DecodeArgs d;
    const uint8_t *k8, *v8;   // as in Store8Args
    const float *scales;
    const uint16_t *open;
    const int32_t *open_slot; // device [n_seqs]: each sequence's open block after the step
};
hipError_t launch_decode8(const Decode8Args &a, hipStream_t s);
// Rows as FP16, from an FP16 cache (k8 null) or an 8-bit one.  What is read
// travels in the arguments: a copy to the device in front of each read would
// cost more than a small read itself.
constexpr int kReadSeqs = 64;  // ranges of a launch, at most
struct ReadRange {
    int32_t seq, first, count;  // rows [first, first + count), count > 0
    int32_t slot;               // the open block that holds its last page (-1: none)
    int32_t open_page;          // and that page
    int32_t to;                 // its first row's place among the output's
    int32_t touch0;             // pages of earlier ranges
};
struct ReadRowsArgs {
    ReadRange range[kReadSeqs];
    int32_t n_ranges;
    int32_t n_touch;            // pages of all ranges
    int32_t num_kv_heads;
    const int32_t *table;
    int32_t table_stride;
    const uint16_t *k_pool, *v_pool;
    const uint8_t *k8, *v8;
    const float *scales;
    const uint16_t *open;
    uint16_t *k_out, *v_out;  // [rows][Hkv][256]
};
hipError_t launch_read_rows(const ReadRowsArgs &a, hipStream_t s);
// Open blocks from their pages' codes, in every layer (bases of layer 0).
struct ReopenArgs {
    const int32_t *touch;     // device [n][kTouchWords]: sequence, page, .., open block
    const int32_t *table;
    int32_t table_stride;
    const uint8_t *k8, *v8;
    const float *scales;
    uint16_t *open;
    size_t layer_codes, layer_scales, layer_open;  // elements between layers
};
hipError_t launch_reopen(const ReopenArgs &a, int32_t n, int32_t num_kv_heads, int32_t n_layers, hipStream_t s);

// ---- eviction (k_evict.hip) ----

constexpr int kMaxObserved = 32;     // query tokens per sequence that kva_attn_weights looks at, at most
// Tiles of 16 query rows (tokens x heads of a group) that a kernel is built for.
constexpr int weight_tiles(int rows) {
    const int t = (rows + 15) / 16;
    return t <= 2 ? t : t <= 4 ? 4 : t <= 8 ? 8 : t <= 12 ? 12 : 16;
}
// Workgroups of it that a CU is given: what LDS (8 KB a tile) and registers hold;
// with one tile three (64 sequences of 16000 rows in 8 bits 266 us; with four 284,
// with two 275).
constexpr int weight_wgs_per_cu(int tiles) { return tiles <= 1 ? 3 : tiles <= 2 ? 3 : tiles <= 4 ? 2 : 1; }
struct WeightArgs {
    const uint16_t *q;        // [T][H][256]
    const int32_t *seq_ids;   // device, as in MultiQueryArgs
    const int32_t *ctx_lens;
    const int32_t *tok_off;
    const int32_t *pre_seq;   // device [n_seqs + 1]: pages of earlier sequences
    const int32_t *table;
    int32_t table_stride;
    const uint16_t *k_pool;   // FP16 cache
    const uint8_t *k8;        // 8-bit cache (null: FP16); v8 unused
    const uint8_t *v8;
    const float *scales;
    const uint16_t *open;
    const int32_t *open_slot; // device [n_seqs] (8-bit cache)
    int32_t n_seqs, num_heads, num_kv_heads;
    int32_t n_obs;
    int32_t chunk;            // pages of a workgroup
    int32_t n_chunks;         // of all sequences
    int32_t part_rows;        // query rows at most
    float2 *part;             // [n_chunks][Hkv][part_rows]: max (log2 units), sum
    float *scores;            // [pages][Hkv][part_rows][16], or null: K is read again
    float decay;
    float *weights;           // [n_seqs][Hkv][w_stride]
    int64_t w_stride;
};
hipError_t launch_weights(const WeightArgs &a, hipStream_t s);

constexpr int kSelectLds = 32768;    // rows whose keys select_kernel holds in LDS, at most
constexpr int kSelectSeqs = 64;      // sequences of a launch, at most (their sizes travel in its arguments)
struct SelectArgs {
    int32_t rows[kSelectSeqs], keep[kSelectSeqs];  // of sequence b0 + i: rows, rows that stay
    int32_t b0, n_seqs;       // of the call
    const float *weights;     // [layers][n_seqs][Hkv][w_stride]
    float *weights_out;       // nullable
    int64_t w_stride;
    int32_t *kept;            // [layers][n_seqs][Hkv][kept_stride]
    int64_t kept_stride;
    int32_t num_kv_heads;
    int32_t first, recent;
};
// n: sequences of the launch; most: rows of the longest.
hipError_t launch_select(const SelectArgs &a, int32_t n, int32_t n_layers, int32_t most, hipStream_t s);

struct GatherArgs {
    // Device [n][kTouchWords]: sequence's index in the call, destination page,
    // source sequence, destination block (of an 8-bit cache's last page, not
    // full: -1 - its open block), rows, the source's open page (-1: none) and
    // open block.
    const int32_t *recs;
    const int32_t *kept;
    int64_t kept_stride;
    int32_t n_seqs;           // of the call
    const int32_t *table;
    int32_t table_stride;
    uint16_t *k_pool, *v_pool;  // layer 0
    size_t layer_elems;
    uint8_t *k8, *v8;
    float *scales;
    uint16_t *open;
    size_t layer_codes, layer_scales, layer_open;
};
hipError_t launch_gather(const GatherArgs &a, int32_t n_recs, int32_t num_kv_heads, int32_t n_layers, hipStream_t s);

}  // namespace kva
