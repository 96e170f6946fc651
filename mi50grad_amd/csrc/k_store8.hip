// Rows into and out of the 8-bit cache (page order, scales and codes:
// k_page8.h), and out of the FP16 one.
//
// Append: each row is what the FP16 cache would hold (norm_rope_apply, the
// same bits).  A step touches pages; a touch and a KV head are one workgroup,
// a half-wave per row of the page.  Where the step brings the page's last row,
// the workgroup takes the rows that came earlier from the sequence's open
// block and writes the page's codes: from FP16 rows always, so a page's codes do
// not depend on the steps that its rows came in.  Otherwise the new rows join
// the open block.  A page that is open after another lies in the sequence's other
// open block, so nothing that a step reads is written by it: its workgroups
// need no order, and an append that is called again gives the same.  Query rows
// are normalised by further workgroups of the launch.
//
// Bound by latency: a decode step's touch is one row (5.5 us for 32 sequences); a
// prompt's workgroups each wait in turn for their rows, three barriers and their
// stores, 1.7 rounds of them for 7000 tokens (43 MB read and written, 17 us where
// a copy takes 9).  LDS is busy for 5 of the 17, over half of that in bank
// conflicts of V's codes, which go there one byte at a time.  Read back 10 us.
#include "k_common.h"
#include "k_normrope.h"
#include "k_page8.h"
#include "kva_internal.h"

namespace kva {
namespace {

constexpr int kThreads = 32 * kBlockTokens;  // a half-wave per row

__global__ __launch_bounds__(kThreads) void store8_kernel(Store8Args a) {
    const AppendArgs &ap = a.ap;
    __shared__ CloseLds lds;
    const int hkv = ap.num_kv_heads, nh = ap.num_heads;
    const int row = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const int n_kv = a.n_touch * hkv;
    if (static_cast<int>(blockIdx.x) >= n_kv) {  // query rows
        const int64_t r = static_cast<int64_t>(blockIdx.x - n_kv) * kBlockTokens + row;
        if (r >= static_cast<int64_t>(ap.n_tok) * nh) return;
        const int t = static_cast<int>(r / nh);
        uint16_t *q = ap.q + r * kHeadDim + 8 * l32;
        const int pos = ap.tok_pos[t];
        const NormRopeIn in = norm_rope_in<32>(ap.q_w, ap.cos_tab + static_cast<size_t>(pos) * ap.half_rot,
                                               ap.sin_tab + static_cast<size_t>(pos) * ap.half_rot, ap.half_rot, l32);
        st16(q, norm_rope_apply<32>(ld16(q), in, ap.half_rot, ap.eps, l32));
        return;
    }
    const int u = blockIdx.x / hkv, h = blockIdx.x - u * hkv;
    const int32_t *rec = a.touch + static_cast<size_t>(u) * kTouchWords;
    const int seq = ld_uniform(rec), page = ld_uniform(rec + 1), tok0 = ld_uniform(rec + 2);
    const int r0 = ld_uniform(rec + 3), n = ld_uniform(rec + 4), slot = ld_uniform(rec + 5);
    const bool closes = r0 + n == kBlockTokens;  // uniform over the workgroup
    uint16_t *open = a.open + (static_cast<size_t>(slot) * hkv + h) * 2 * kPageElems;
    const bool fresh = row >= r0 && row < r0 + n;
    const int t = fresh ? tok0 + row - r0 : 0;
    const size_t at = (static_cast<size_t>(t) * hkv + h) * kHeadDim + 8 * l32;
    BlockRow x{};
    if (fresh) {
        x.k = ld16(ap.k + at);
        x.v = ld16(ap.v + at);
    } else if (closes) {  // row < r0
        x = load_open_row(open, row, l32);
    }
    if (a.norm) {  // by every half-wave, so that its lane exchanges are whole
        const int pos = fresh ? ap.tok_pos[t] : 0;
        const NormRopeIn in = norm_rope_in<32>(ap.k_w, ap.cos_tab + static_cast<size_t>(pos) * ap.half_rot,
                                               ap.sin_tab + static_cast<size_t>(pos) * ap.half_rot, ap.half_rot, l32);
        const uint4 y = norm_rope_apply<32>(x.k, in, ap.half_rot, ap.eps, l32);
        if (fresh) {
            x.k = y;
            if (!ap.keep_k) st16(ap.k + at, y);
        }
    }
    mend_row(x);  // an earlier row of the open block has been through this
    if (!closes) {
        if (fresh) store_open_row(open, row, l32, x);
        return;
    }
    const int blk = ld_uniform(ap.table + static_cast<size_t>(seq) * ap.table_stride + page);
    const size_t b = static_cast<size_t>(blk) * hkv + h;
    close_block(x, a.k8 + b * kPageElems, a.v8 + b * kPageElems, a.scales + 2 * b, lds);
}

// Rows of both kinds of cache as FP16 [row][Hkv][256]; a page of a range and a
// KV head per workgroup.
template <bool kInt8>
__global__ __launch_bounds__(kThreads) void read_rows_kernel(ReadRowsArgs a) {
    const int hkv = a.num_kv_heads;
    const int row = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const int u = blockIdx.x / hkv, h = blockIdx.x - u * hkv;
    // The range: the last whose pages begin at or before this one (each has some).
    static_assert(kReadSeqs == 64, "a range per lane");
    const int lane = threadIdx.x & 63;
    const uint64_t before = __ballot(lane < a.n_ranges && a.range[lane].touch0 <= u);
    const ReadRange &g = a.range[__builtin_amdgcn_readfirstlane(63 - __clzll(before))];
    const int seq = g.seq, slot = g.slot;
    const int page = (g.first >> 4) + u - g.touch0;
    const int from = max(g.first, 16 * page), r0 = from & 15;
    const int n = min(g.first + g.count, 16 * page + 16) - from;
    const int to = g.to + from - g.first;
    const bool is_open = kInt8 && slot >= 0 && page == g.open_page;
    const bool mine = row >= r0 && row < r0 + n;
    const int blk = is_open ? 0 : ld_uniform(a.table + static_cast<size_t>(seq) * a.table_stride + page);
    BlockRow x{};
    if constexpr (kInt8) {
        __shared__ __attribute__((aligned(16))) uint8_t codes[2][kPageElems];
        if (is_open) {
            if (mine)
                x = load_open_row(a.open + (static_cast<size_t>(slot) * hkv + h) * 2 * kPageElems, row, l32);
        } else {
            const size_t b = static_cast<size_t>(blk) * hkv + h;
            reinterpret_cast<uint2 *>(codes[0])[threadIdx.x] =
                reinterpret_cast<const uint2 *>(a.k8 + b * kPageElems)[threadIdx.x];
            reinterpret_cast<uint2 *>(codes[1])[threadIdx.x] =
                reinterpret_cast<const uint2 *>(a.v8 + b * kPageElems)[threadIdx.x];
            __syncthreads();
            x = load_code_row(codes[0], codes[1], a.scales + 2 * b, row, l32);
        }
    } else if (mine) {
        const size_t at = ((static_cast<size_t>(blk) * kBlockTokens + row) * hkv + h) * kHeadDim + 8 * l32;
        x.k = ld16(a.k_pool + at);
        x.v = ld16(a.v_pool + at);
    }
    if (!mine) return;
    const size_t at = (static_cast<size_t>(to + row - r0) * hkv + h) * kHeadDim + 8 * l32;
    st16(a.k_out + at, x.k);
    st16(a.v_out + at, x.v);
}

// Rows as they are into the FP16 pool (append_rows): a half-wave per row of a head.
__global__ __launch_bounds__(256) void copy_rows_kernel(AppendArgs a) {
    const int l32 = threadIdx.x & 31;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int hkv = a.num_kv_heads;
    if (r >= static_cast<int64_t>(a.n_tok) * hkv) return;
    const int t = static_cast<int>(r / hkv), h = static_cast<int>(r - static_cast<int64_t>(t) * hkv);
    const int slot = a.tok_slot[t];
    const int blk = a.table[static_cast<size_t>(a.tok_seq[t]) * a.table_stride + (slot >> 4)];
    const size_t at = ((static_cast<size_t>(blk) * kBlockTokens + (slot & 15)) * hkv + h) * kHeadDim + 8 * l32;
    st16(a.k_pool + at, ld16(a.k + r * kHeadDim + 8 * l32));
    st16(a.v_pool + at, ld16(a.v + r * kHeadDim + 8 * l32));
}

// The open blocks of sequences whose length was set back into a full page:
// that page's values, in FP16.  grid (record, KV head, layer).
__global__ __launch_bounds__(kThreads) void reopen_kernel(ReopenArgs a) {
    const int hkv = gridDim.y, h = blockIdx.y, layer = blockIdx.z;
    const int32_t *rec = a.touch + static_cast<size_t>(blockIdx.x) * kTouchWords;
    const int seq = ld_uniform(rec), page = ld_uniform(rec + 1), slot = ld_uniform(rec + 5);
    const int blk = ld_uniform(a.table + static_cast<size_t>(seq) * a.table_stride + page);
    const size_t b = static_cast<size_t>(blk) * hkv + h;
    const float2 s = *reinterpret_cast<const float2 *>(a.scales + layer * a.layer_scales + 2 * b);
    uint16_t *open = a.open + layer * a.layer_open + (static_cast<size_t>(slot) * hkv + h) * 2 * kPageElems;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const uint8_t *codes = (kv ? a.v8 : a.k8) + layer * a.layer_codes + b * kPageElems;
        const uint2 c = reinterpret_cast<const uint2 *>(codes)[threadIdx.x];
        const uint32_t s2 = scale_h2(kv ? s.y : s.x);
        const uint2 lo = values4(c.x, s2), hi = values4(c.y, s2);
        st16(open + kv * kPageElems + 8 * threadIdx.x, make_uint4(lo.x, lo.y, hi.x, hi.y));
    }
}

}  // namespace

hipError_t launch_store8(const Store8Args &a, hipStream_t s) {
    if (a.ap.n_tok <= 0) return hipSuccess;
    const int64_t q_rows = a.norm ? static_cast<int64_t>(a.ap.n_tok) * a.ap.num_heads : 0;
    const int64_t wgs = static_cast<int64_t>(a.n_touch) * a.ap.num_kv_heads + (q_rows + kBlockTokens - 1) / kBlockTokens;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(store8_kernel, dim3(static_cast<unsigned>(wgs)), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_copy_rows(const AppendArgs &a, hipStream_t s) {
    const int64_t wgs = (static_cast<int64_t>(a.n_tok) * a.num_kv_heads + 7) / 8;
    if (wgs <= 0) return hipSuccess;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(copy_rows_kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_read_rows(const ReadRowsArgs &a, hipStream_t s) {
    const int64_t wgs = static_cast<int64_t>(a.n_touch) * a.num_kv_heads;
    if (wgs <= 0) return hipSuccess;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(wgs));
    if (a.k8)
        hipLaunchKernelGGL(read_rows_kernel<true>, grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL(read_rows_kernel<false>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_reopen(const ReopenArgs &a, int32_t n, int32_t num_kv_heads, int32_t n_layers, hipStream_t s) {
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(reopen_kernel, dim3(n, num_kv_heads, n_layers), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace kva
