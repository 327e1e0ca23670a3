// Rows into pages of the e4m3 layout with K through RMSNorm and the rotary first (launched in f8p_move.hip, with a rotary of several
// axes in f8p_axes.hip).
#pragma once

#include "f8p_rows.hpp"

namespace bkv {

namespace {

// The same with K through RMSNorm and the rotary first; arithmetic as in append_kprep_kernel (kv_move.hip).  A work-group has both
// halves of a (page, kv head): V arrives, is coded and stored while one wave adds up K's squares, one after the other as the sum
// is defined.  Eight work-groups a compute unit, as many as LDS and threads let be there, hide what they can of that chain
// (registers are kept to that: 86 of them and five work-groups cost two prompts of 8191 tokens 3 us).  Those, 84 MB, take 21.7 us;
// without the sums, the products and the rotary, 17 us.
struct F8Prep {
    const float* gamma;
    const float* table;
    const int32_t* positions;
    float eps;
    int32_t n_rot, max_pos;
};
constexpr int kPrepStride = kF8Hd + 4;
// AXES: the position of a pair is that of the token on the pair's axis.  2073 tokens of 4 kv heads, 64 pairs: 13.1 us, 12.4 with one position
// a cell.  Five work-groups a compute unit, all there at once: the chain of trips and barriers that each goes through.  Of the 13.1, with
// the squares of four elements in place of 256 11.0, with one pair in place of 64 11.7, with both 9.3; rows that stay in their pages cost
// nothing that shows (13.2 without).
struct F8PrepAxes : F8Prep {
    KPrepAxes axes;
};
template <typename Batch, bool AXES>
__global__ __launch_bounds__(kBlock, 8) void append_kprep_f8p_kernel(Batch b, F8MoveGeom g, std::conditional_t<AXES, F8PrepAxes, F8Prep> kp, uint8_t* __restrict__ kpool,
                                                                     uint8_t* __restrict__ vpool, const int32_t* __restrict__ tables,
                                                                     const float* __restrict__ ks, const float* __restrict__ vs) {
#pragma clang fp contract(off)
    __shared__ float red_v[kF8Waves], red_k[kF8Waves];
    __shared__ __attribute__((aligned(16))) float rows_s[kF8Page * kPrepStride];
    __shared__ double inv_s[kF8Page];
    int at_page = (int)blockIdx.x / g.n_kv;
    const int kvh = (int)blockIdx.x - at_page * g.n_kv;
    F8Rows r;
    if (!find(b, at_page, r)) return;
    const F8Span s = span_of(r, at_page);
    const int tid = threadIdx.x;
    const F8Share at(tid);
    const F8Target t = target_of(g, kpool, vpool, tables, r.row, s.page, kvh);
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x[4];
        load4(ks + source_of(r, s, g.n_kv, kvh, at.v_row + i, at.v_col), x);
        *reinterpret_cast<float4*>(rows_s + (at.v_row + i) * kPrepStride + at.v_col) = make_float4(x[0], x[1], x[2], x[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) load4(vs + source_of(r, s, g.n_kv, kvh, at.v_row + i, at.v_col), v[i]);
    const float gamma = kp.gamma[tid];
    F8Old old{};
    if (s.kept > 0) old = old_of<true>(t, at);
    __syncthreads();
    // (one wave of the four, another in the next work-group: a compute unit's would all wait for one SIMD: 0.7 us of the prompts')
    const int sum_row = (tid ^ (int)(blockIdx.x << 6)) & (kBlock - 1);
    if (sum_row < kF8Page) {
        double ss = 0.0;  // in element order; a product of two floats is exact, fused it is the same sum
#pragma unroll 4
        for (int i = 0; i < kF8Hd; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(rows_s + sum_row * kPrepStride + i);
            ss = __builtin_fma((double)x.x, (double)x.x, ss);
            ss = __builtin_fma((double)x.y, (double)x.y, ss);
            ss = __builtin_fma((double)x.z, (double)x.z, ss);
            ss = __builtin_fma((double)x.w, (double)x.w, ss);
        }
        inv_s[sum_row] = 1.0 / sqrt(ss / (double)kF8Hd + (double)kp.eps);
    }
    settle_rows<true>(at, v, s.kept, s.end, old, red_v, tid);
    __syncthreads();
    store_codes<true>(at, v, red_v, t.vunit, t.line + 1, tid);
#pragma unroll 4
    for (int row = 0; row < kF8Page; ++row) {
        float* d = rows_s + row * kPrepStride + tid;
        *d = (float)((double)*d * inv_s[row] * (double)gamma);
    }
    __syncthreads();
    // the rotary: pairs tid / 16 + 16 i of row tid % 16 (clamped to the call's cells: positions need not cover others)
    const int half = kp.n_rot / 2, rot_row = tid & (kF8Page - 1);
    const int cell = min(max(s.page * kF8Page + rot_row, r.pos0), r.pos0 + r.n_tok - 1);
    int pos = 0;
    if constexpr (!AXES) pos = min(max(kp.positions ? kp.positions[cell] : cell, 0), kp.max_pos - 1);
    const float2* const factors = reinterpret_cast<const float2*>(kp.table) + (size_t)pos * half;
    float* const d = rows_s + rot_row * kPrepStride;
    for (int j = tid / kF8Page; j < half; j += kBlock / kF8Page) {
        float2 cs;
        if constexpr (AXES) cs = factors[(size_t)axis_position(kp.axes, j, (size_t)(r.src0 + (cell - r.pos0)), kp.max_pos) * half + j];
        else cs = factors[j];
        const double x = (double)d[j], y = (double)d[j + half], c = (double)cs.x, si = (double)cs.y;
        const double xc = x * c, ys = y * si, xs = x * si, yc = y * c;
        d[j] = (float)(xc - ys);
        d[j + half] = (float)(xs + yc);
    }
    __syncthreads();
    float k[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(rows_s + at.k_row * kPrepStride + at.k_col + 32 * u);
        k[u][0] = x.x, k[u][1] = x.y, k[u][2] = x.z, k[u][3] = x.w;
    }
    if (s.kept > 0) old = old_of<false>(t, at);
    settle_rows<false>(at, k, s.kept, s.end, old, red_k, tid);
    __syncthreads();
    store_codes<false>(at, k, red_k, t.kunit, t.line, tid);
}

}  // namespace

}  // namespace bkv
