// What the attention kernels over e4m3 pages (f8p.hpp) share: the mathematics, for a wave that walks pages two at a time with tiles
// of 16 query rows.
//
//   S^T[cell][row] = K[cell][:] . Q[row][:]      v_mfma_f32_16x16x32_f16, A = K (codes as f16, exact), B = q
//   z              = S^T * 2^(e_K) + e_V          base-2 logits plus the exponent of the page's V
//   w              = exp2(z - M)                  M: kF8Lift below a running maximum of z, moved when that is passed by more than kF8Slack
//   O^T[d][row]   += V^T[d][cell] . w[cell][row]  A = V (codes as f16, exact), 32 cells of two pages a product
//   l             += w * 2^(-e_V)
//
// So the scale of K is a factor of the page's scores and that of V rides on the weights: the largest terms have the largest weights
// whatever the magnitude of their values, pages of different scales meet in one product, and out = O / l with both relative to
// M.  Exponents lie in -32 .. 31, which keeps the terms of l below 2^(kF8Lift + kF8Slack + 32 + log2 of the cells) and its largest one
// at 2^(kF8Lift - 31) or more.
//
// q and the weights enter as the sum of two f16 numbers (two products each).  q's row is brought to a largest value of 2^13 .. 2^14 first,
// by a power of two that rejoins the scale of K: neither part leaves what f16 can hold, whatever the queries' size, and an element is
// off by 2^-22 of itself and 2^-38 of the row's largest.  A weight is off by 2^-22 of itself or by 2^-25: f16's steps end there.
// The largest term's is 2^kF8Lift .. 2^(kF8Lift + kF8Slack), as far up as f16 reaches, so a term is off by 2^-22 of itself and 2^-34
// of the largest one.  (M at the maximum itself made the latter 2^-25: a chunk's 8000 equal weights behind a key that brings nothing,
// 19.7 bits above them, were off by 1.5e-2 of the output, 25.6 bits above them they were lost; now 7e-5 and 6e-4, in the same
// time.)  The sums are f32, in the matrix cores.
//
// A lane (c = lane % 16, g = lane / 16) holds of a tile row c, and cells 4 g .. 4 g + 3 of either page: weights come out of the
// softmax in the order the second product takes them in.
#pragma once

#include <hip/hip_runtime.h>

#include "f8p.hpp"
#include "lane_groups.hpp"

namespace bkv {

typedef _Float16 f8_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 f8_h2 __attribute__((ext_vector_type(2)));
typedef float f8_f4 __attribute__((ext_vector_type(4)));

constexpr float kF8Lift = 9.0f, kF8Slack = 6.0f;  // 2^15 at most: f16 ends at 65504
// Where M goes when it moves to a maximum.  (From 2^24 on f32 does not hold what lies kF8Lift below: from 2^27 it would be 16 below, and
// weights past f16's end.)
__device__ __forceinline__ float f8_reference(float top) {
    const float at = top - kF8Lift;
    return top - at > kF8Lift + kF8Slack ? top : at;
}

// 2^up for the elements of a row of q; NaN where the scale of the logits is not finite.  (Where that scale is used it is kept
// finite, and a NaN would not come through.)
__device__ __forceinline__ float f8_lift_q(int up, float scale_log2e) { return exp2_int(up) + (scale_log2e - scale_log2e); }

__device__ __forceinline__ f8_f4 f8_mfma(f8_h8 a, f8_h8 b, f8_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// 4 + 4 codes as f16 numbers; the conversion is exact (e4m3's subnormals are f16 normals), NaN stays NaN
__device__ __forceinline__ f8_h8 f8_to_f16(unsigned a, unsigned b) {
    const f8_h2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, true);
    const f8_h2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, true);
    return f8_h8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

}  // namespace bkv
