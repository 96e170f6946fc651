// The stream-K walk of a decode launch: the pages of every sequence laid end
// to end, shared out among workgroups, and a cursor over a share's pages.
#pragma once

#include "k_common.h"
#include "kva_internal.h"

namespace kva {

__device__ __forceinline__ const uint16_t *gate_of(const DecodeArgs &a, int b, int hq, int lane) {
    return a.gate ? a.gate + static_cast<int64_t>(b) * a.gate_stride + hq * kHeadDim + 4 * lane : nullptr;
}

// First page of workgroup w when P pages are shared by W workgroups.
// kFast: floor_muldiv's 32-bit division when the product fits, for the
// combine, which waits on these before its first loads; the decode kernel
// keeps the 64-bit form (the extra branch cost it registers: one wave per
// SIMD instead of two, C3 114 -> 144 us).
template <bool kFast = false>
__device__ __forceinline__ int wg_start(int w, int P, int W) {
    return kFast ? floor_muldiv(w, P, W) : static_cast<int>(static_cast<int64_t>(w) * P / W);
}

// The workgroup whose page range holds page p.
template <bool kFast = false>
__device__ __forceinline__ int wg_of_page(int p, int P, int W) {
    int w = kFast ? floor_muldiv(p, W, P) : static_cast<int>(static_cast<int64_t>(p) * W / P);
    while (w + 1 < W && wg_start<kFast>(w + 1, P, W) <= p) ++w;
    return w;
}

// The stream-K shape of a launch: P pages over W workgroups.  Fixed by the
// host for an ordinary call; for a launch recorded into a graph it is derived
// here from the step plan (the same rule the host applies), so a replay after
// the lengths grew still shares the right page count.
__device__ __forceinline__ void stream_k_shape(const DecodeArgs &a, int &P, int &W) {
    if (!a.dyn) {
        P = a.total_pages;
        W = a.n_wg;
        return;
    }
    P = ld_uniform(a.pre_seq + a.n_seqs);
    int w = a.split_tokens > 0 ? (P * kBlockTokens + a.split_tokens - 1) / a.split_tokens : a.n_wg;
    w = min(w, (P + a.min_pages - 1) / a.min_pages);
    W = max(1, min(w, a.n_wg));
}

// Pages of all sequences before sequence b.
__device__ __forceinline__ int seq_page_base(const DecodeArgs &a, int b, int npg) {
    return a.pre_seq ? a.pre_seq[b] : b * npg;
}

// Per-sequence facts for sequences b0 .. b0+63, one per lane, so a sequence
// switch costs v_readlane instead of a chain of dependent loads.
struct SeqWindow {
    int b0;
    int base, ctx, sid;  // this lane's sequence: first page, length, cache slot
};

__device__ __forceinline__ void load_window(SeqWindow &win, const DecodeArgs &a, int b0, int lane) {
    const int i = b0 + lane;
    const bool ok = i < a.n_seqs;
    const int npg_c = (a.ctx_len_const + 15) >> 4;
    win.b0 = b0;
    win.ctx = ok ? (a.ctx_lens ? a.ctx_lens[i] : a.ctx_len_const) : 0;
    win.base = ok ? (a.pre_seq ? a.pre_seq[i] : i * npg_c) : INT32_MAX;  // lanes past n_seqs: unused
    win.sid = (ok && a.table) ? a.seq_ids[i] : 0;
}

// A page of the workgroup's range: sequence b (index in the step), page pg of
// it.  Every field is wave-uniform.
struct Cursor {
    int b, pg, npg, ctx, base, sid;
    bool ok;
};

__device__ __forceinline__ Cursor seq_cursor(const SeqWindow &win, int b) {
    Cursor c;
    const int k = b - win.b0;
    c.b = b;
    c.pg = 0;
    c.ctx = __builtin_amdgcn_readlane(win.ctx, k);
    c.base = __builtin_amdgcn_readlane(win.base, k);
    c.sid = __builtin_amdgcn_readlane(win.sid, k);
    c.npg = (c.ctx + 15) >> 4;
    c.ok = true;
    return c;
}

}  // namespace kva
